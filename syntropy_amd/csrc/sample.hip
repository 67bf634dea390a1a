// A token of each row of logits x [rows][vocab] by temperature T, top-k, top-p, min-p and a given u in [0, 1).
// The row's logits in order (descending, the lower index first among equals), w_i = exp((x_i - max x) / T):
//   top-k keeps the first k; top-p the least n of those whose sum of w reaches p times theirs; min-p those with
//   w_i >= min_p.  Each keeps a first part of the order, so all together do: n values, of the sum W.
//   The token is the first of them whose running sum passes u W.
// T = 0 stands for top-k 1.
//
// A token and a count are whole numbers, and the borders between tokens are as near to one another as 1e-6 of W, so
// sums are exact to about 2^-44 of a weight whatever their order: with t_i = (max x - x_i) log2(e) / T in 64 bits,
// values are put in bins of 1/32 of t, and a bin's weights are added as whole numbers of 2^-(bits) of the weight
// in the bin's middle.  A bin is a run of the order; a prefix of the order is whole bins, whose sums are
// added in 64 bits in their order, and a part of one.
//
// The row is read three times: for its greatest value, for the bins, and for the few values that a border or the
// token can lie among, which are put in order as a list.  With a top-k (of at most LIST) the bins are counts of F32
// distances, and the list all that can count; with min-p alone no bins are needed.  Only equal values by the thousand
// make more of a bin than a list holds: then a border is found digit by digit of the values' keys.
// Few long rows are split over workgroups, a launch a step.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace syn {

namespace {

constexpr int SB = 2048;        // bins; the last one holds all that is below 2^-64 too (as nothing)
constexpr int ST = 1024;        // threads a workgroup
constexpr uint32_t KEY_INF = 0xFF800000u, KEY_NONE = 0x007FFFFFu;  // sp_order of +-infinity

// A whole number that orders as the value does (-0 as +0, every NaN above +infinity).
SYN_DEV uint32_t sp_order(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = f2u(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
SYN_DEV float sp_value(uint32_t k) { return u2f(k >> 31 ? k ^ 0x80000000u : ~k); }

template <int TY>
SYN_DEV float sp_load(const uint8_t* row, int64_t i) {
    if constexpr (TY == T_F32) return ((const float*)row)[i];
    const uint32_t h = ((const uint16_t*)row)[i];
    return TY == T_F16 ? f16_to_f32(h) : u2f(h << 16);
}

// 2^(-j / 32): what a whole number of bin 32 i + j stands for is 2^-i of it, by the scale's 2^bits.
__constant__ const double STEPS[32] = {
    0x1.0000000000000p+0, 0x1.f50765b6e4540p-1, 0x1.ea4afa2a490dap-1, 0x1.dfc97337b9b5fp-1, 0x1.d5818dcfba487p-1,
    0x1.cb720dcef9069p-1, 0x1.c199bdd85529cp-1, 0x1.b7f76f2fb5e47p-1, 0x1.ae89f995ad3adp-1, 0x1.a5503b23e255dp-1,
    0x1.9c49182a3f090p-1, 0x1.93737b0cdc5e5p-1, 0x1.8ace5422aa0dbp-1, 0x1.82589994cce13p-1, 0x1.7a11473eb0187p-1,
    0x1.71f75e8ec5f74p-1, 0x1.6a09e667f3bcdp-1, 0x1.6247eb03a5585p-1, 0x1.5ab07dd485429p-1, 0x1.5342b569d4f82p-1,
    0x1.4bfdad5362a27p-1, 0x1.44e086061892dp-1, 0x1.3dea64c123422p-1, 0x1.371a7373aa9cbp-1, 0x1.306fe0a31b715p-1,
    0x1.29e9df51fdee1p-1, 0x1.2387a6e756238p-1, 0x1.1d4873168b9aap-1, 0x1.172b83c7d517bp-1, 0x1.11301d0125b51p-1,
    0x1.0b5586cf9890fp-1, 0x1.059b0d3158574p-1};

// The scale of a row's distances and of its weights.
struct Scale {
    double m, c;  // the greatest logit; 32 log2(e) / T
    double one;   // 2^bits: the whole number of a bin's middle weight
    int bits;
    // 32 t of a value
    SYN_DEV double s(float x) const { return (m - (double)x) * c; }
    static SYN_DEV int bin(double s) { return s < (double)(SB - 1) ? (int)__builtin_rint(s) : SB - 1; }
    // the weight of s as a whole number in its bin: 2^(-(s - bin) / 32), |s - bin| <= 1/2 (and where s is 0 exactly 1, so
    // that equal logits have borders where they are to have them)
    SYN_DEV uint64_t whole(double s, int b) const {
        if (!(s < (double)SB)) return 0;
        const double y = (s - (double)b) * (-0.69314718055994530942 / 32.0);
        double p = __builtin_fma(y, 1.0 / 120.0, 1.0 / 24.0);
        p = __builtin_fma(p, y, 1.0 / 6.0);
        p = __builtin_fma(p, y, 0.5);
        p = __builtin_fma(p, y, 1.0);
        p = __builtin_fma(p, y, 1.0);
        // (below 2^51: added to 2^52 its whole part is the sum's last bits)
        return __builtin_bit_cast(uint64_t, __builtin_fma(p, one, 0x1p52)) & 0xFFFFFFFFFFFFFull;
    }
    SYN_DEV double weight(double s) const { return exp2(s * (-1.0 / 32.0)); }
    // what a whole number of bin b stands for
    SYN_DEV double unit(int b) const { return ldexp(STEPS[b & 31], -(b >> 5) - bits); }
};

enum Want { AT_LEAST_N, SUM_REACHES, SUM_PASSES };

constexpr int LIST = 2048;  // keys that a workgroup sorts

// What a row is asked for, and what follows from its greatest value.
struct Asked {
    bool fit;        // its settings say something
    float u, top_p;
    uint32_t k;      // (all: 2^32 - 1)
    float min_p;
    double last;     // the greatest s that min-p keeps
};

enum Mode { LIST_K, LIST_MIN_P, BINS };  // top-k by counts; min-p alone; the bins' sums

// What is gathered: of LIST_K the F32 bins up to a1, of LIST_MIN_P what min-p keeps, of BINS those from a0 to a1 and b.
struct Wanted {
    int a0, a1, b;   // (b: none where negative)
    int cut;         // BINS: the bin of the border (none: -1)
    bool by_p, by_min_p;
    uint32_t n;      // how many values that is
};

// Where bin b lies: neighbours in different banks, and so the 64 octaves of 32 bins, a lane each.
SYN_DEV int sp_at(int b) { return (b & 31) * 65 + (b >> 5); }
constexpr int SLOTS = 32 * 65;  // (bin SB, the end, lies at 64)

struct Row {
    uint32_t counts[SLOTS];      // of a bin's values, then of those before it
    uint64_t masses[SLOTS];      // of a bin, then (as double) the sum before it
    alignas(16) uint64_t keys[LIST];  // the gathered values' keys: (order from above, index), so that they order upwards
    double run[LIST];         // the running sum at each, from the row's first value on
    double part[ST / 64];
    uint32_t most, at, n;
    int bin;
    Wanted want;
    // of descend()
    uint64_t prefix, before_mass;
    uint32_t before;
    double sum;
    SYN_DEV uint32_t count0(int b) const { return counts[sp_at(b)]; }
    SYN_DEV double base(int b) const { return __builtin_bit_cast(double, masses[sp_at(b)]); }
    SYN_DEV uint32_t in(int b) const { return count0(b + 1) - count0(b); }
};

SYN_DEV uint64_t sp_key(float v, int i) { return (uint64_t)~sp_order(v) << 32 | (uint32_t)i; }
SYN_DEV float sp_of_key(uint64_t k) { return sp_value(~(uint32_t)(k >> 32)); }

// A place in the order: how many values reach it, their sum, and the key of the last one.
struct Place {
    uint32_t n;
    double sum;
    uint64_t key;
};

template <int TY>
struct Sampler {
    static constexpr int PER = TY == T_F32 ? 4 : 8, ES = TY == T_F32 ? 4 : 2;
    const uint8_t* x;
    int vocab;
    Row& r;
    Scale sc{};
    Asked q{};
    int first_piece = 0, end_piece = 0;  // of 16 bytes, this workgroup's part (the row's last values are the last part's)

    SYN_DEV Sampler(const SampleArgs& g, uint64_t row, Row& rr) : x((const uint8_t*)g.x + row * g.ldx * ES), vocab(g.vocab), r(rr) {
        const float t = g.temperature ? g.temperature[row] : g.temperature0;
        const int k = g.top_k ? g.top_k[row] : g.top_k0;
        q.top_p = g.top_p ? g.top_p[row] : g.top_p0;
        q.min_p = g.min_p ? g.min_p[row] : g.min_p0;
        q.u = g.u[row];
        const bool greedy = t == 0.0f;
        q.fit = (greedy || (t >= 0x1p-64f && t <= 0x1p64f)) && q.top_p == q.top_p && q.min_p == q.min_p && q.u == q.u;
        q.k = greedy ? 1u : k > 0 ? (uint32_t)k : 0xFFFFFFFFu;
        q.u = q.u < 0.0f ? 0.0f : q.u > 0x1.fffffep-1f ? 0x1.fffffep-1f : q.u;
        q.min_p = q.min_p < 1.0f ? q.min_p : 1.0f;
        q.last = q.min_p > 0.0f ? -32.0 * log2((double)q.min_p) : __builtin_inf();
        sc.c = 32.0 * 1.44269504088896340736 / (greedy ? 1.0 : (double)t);
        int bits = 62;
        for (uint32_t v = 1; v < (uint32_t)vocab; v *= 2) --bits;
        sc.bits = bits < 50 ? bits : 50;
        sc.one = ldexp(1.0, sc.bits);
        end_piece = vocab / PER;
    }
    // Part `part` of `parts`.
    SYN_DEV void take(int part, int parts) {
        const int all = vocab / PER;
        first_piece = (int)((int64_t)all * part / parts);
        end_piece = (int)((int64_t)all * (part + 1) / parts);
    }
    // false: the row has no distribution
    SYN_DEV bool set_most(uint32_t most) {
        sc.m = sp_value(most);
        return q.fit && most < KEY_INF && most > KEY_NONE;
    }
    SYN_DEV Mode mode() const {
        return q.k <= (uint32_t)LIST && q.k < (uint32_t)vocab ? LIST_K : q.top_p >= 1.0f && q.min_p > 0.0f && q.k >= (uint32_t)vocab ? LIST_MIN_P : BINS;
    }

    SYN_DEV static float value(const uint32_t (&w)[4], int j) {
        if constexpr (TY == T_F32) return u2f(w[j]);
        const uint32_t h = w[j / 2];
        if constexpr (TY == T_F16) return f16_to_f32(j & 1 ? h >> 16 : h);
        return u2f(j & 1 ? h & 0xFFFF0000u : h << 16);
    }
    // f(value, index) of this workgroup's values, 16 bytes a load, at any value's address.  Four loads are in flight;
    // where f is long they are passed down (moves) to one copy of it, for code that is read once costs its way into
    // the instruction cache: with four copies, and the steps below as often as they are used, a row of 32064 took 15 us.
    template <bool SHORT, class F>
    SYN_DEV void each(F&& f) const {
        constexpr int MANY = 4;
        uint32_t w[MANY][4];
        auto load = [&](int p, uint32_t (&to)[4]) { __builtin_memcpy(to, x + (int64_t)(p < end_piece ? p : first_piece) * 16, 16); };
        auto use = [&](int p, const uint32_t (&from)[4]) {
            if (p >= end_piece) return;
#pragma unroll
            for (int j = 0; j < PER; ++j) f(value(from, j), p * PER + j);
        };
        int p = first_piece + (int)threadIdx.x;
        if (first_piece < end_piece) {
#pragma unroll
            for (int m = 0; m < MANY; ++m) load(p + ST * m, w[m]);
            if constexpr (SHORT) {
                for (; p < end_piece; p += ST * MANY) {
                    uint32_t o[MANY][4];
#pragma unroll
                    for (int m = 0; m < MANY; ++m) __builtin_memcpy(o[m], w[m], 16);
                    if (p + ST * MANY < end_piece) {
#pragma unroll
                        for (int m = 0; m < MANY; ++m) load(p + ST * (MANY + m), w[m]);
                    }
#pragma unroll
                    for (int m = 0; m < MANY; ++m) use(p + ST * m, o[m]);
                }
            } else {
#pragma unroll 1
                for (; p < end_piece; p += ST) {
                    uint32_t o[4];
                    __builtin_memcpy(o, w[0], 16);
#pragma unroll
                    for (int m = 0; m + 1 < MANY; ++m) __builtin_memcpy(w[m], w[m + 1], 16);
                    load(p + ST * MANY, w[MANY - 1]);
                    use(p, o);
                }
            }
        }
        const int i = vocab / PER * PER + (int)threadIdx.x;
        if (i < vocab && end_piece == vocab / PER) f(sp_load<TY>(x, i), i);
    }
    // The same of the whole row, value by value: for what is seldom.
    template <class F>
    SYN_DEV void every(F&& f) const {
#pragma unroll 1
        for (int i = threadIdx.x; i < vocab; i += ST) f(sp_load<TY>(x, i), i);
    }

    // (every thread) the sums over the threads before this one, and all of them
    template <class T>
    SYN_DEV T before(T v, T* part, T& all) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        T s = v;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const T o = __shfl_up(s, d);
            s += lane >= d ? o : T(0);
        }
        if (lane == 63) part[wave] = s;
        __syncthreads();
        T off = 0, sum = 0;
#pragma unroll
        for (int w = 0; w < ST / 64; ++w) {
            off += w < wave ? part[w] : T(0);
            sum += part[w];
        }
        all = sum;
        __syncthreads();
        return off + s - v;
    }

    // (one wavefront) The counts and sums of the bins before each, in place: an octave a lane.
    SYN_DEV void prefix(bool sums) {
        const int l = threadIdx.x & 63;
        uint32_t n = 0;
        double s = 0.0;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            n += r.counts[j * 65 + l];
            if (sums) s = __builtin_fma((double)r.masses[j * 65 + l], STEPS[j], s);
        }
        const double one = ldexp(1.0, -l - sc.bits);
        s *= one;
        uint32_t bn = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t on = __shfl_up(bn, d);
            bn += l >= d ? on : 0u;
        }
        const uint32_t all = __shfl(bn, 63);
        n = bn - n;
        // The sums before each octave one after another, so that they grow exactly where an octave holds something: a
        // border found between two of them is a bin that does.
        double from = 0.0, next = 0.0;
        for (int o = 0; sums && o < 64; ++o) {
            from = l >= o ? next : from;
            if (__shfl(n, o) == all) break;  // uniform: nothing from here on
            next += __shfl(s, o);
        }
        const double end = next;
        double in = 0.0;
#pragma unroll 8
        for (int j = 0; j < 32; ++j) {
            const uint32_t c = r.counts[j * 65 + l];
            r.counts[j * 65 + l] = n;
            n += c;
            if (sums) {
                const double m = (double)r.masses[j * 65 + l];
                r.masses[j * 65 + l] = __builtin_bit_cast(uint64_t, from + in * one);
                in = __builtin_fma(m, STEPS[j], in);
            }
        }
        if (l == 63) r.counts[64] = all, r.masses[64] = __builtin_bit_cast(uint64_t, end);
        wave_lds_sync();
    }
    // (one wavefront) The first bin whose values reach what is wanted (the last that holds any where none does).
    SYN_DEV int bin_of(Want want, uint32_t n, double sum) const {
        const int l = threadIdx.x & 63;
        auto so = [&](int b) {
            return want == AT_LEAST_N ? r.count0(b + 1) >= n : want == SUM_REACHES ? r.base(b + 1) >= sum : r.base(b + 1) > sum;
        };
        uint64_t yes = __builtin_amdgcn_ballot_w64(so(32 * l + 31));
        if (yes == 0) {
            want = AT_LEAST_N, n = r.count0(SB);
            yes = __builtin_amdgcn_ballot_w64(so(32 * l + 31));
        }
        const int o = 32 * (__builtin_ffsll((long long)yes) - 1);
        return o + __builtin_ffsll((long long)__builtin_amdgcn_ballot_w64(l < 32 && so(o + (l & 31)))) - 1;
    }

    // (every thread) the least of the threads' numbers
    SYN_DEV uint32_t least(uint32_t v) {
        if (threadIdx.x == 0) r.at = 0xFFFFFFFFu;
        __syncthreads();
        v = group_min_u32<64>(v);
        if ((threadIdx.x & 63) == 0 && v != 0xFFFFFFFFu) atomicMin(&r.at, v);
        __syncthreads();
        const uint32_t m = r.at;
        __syncthreads();
        return m;
    }
    // The keys that `pick` takes, in order, into r.keys; returns how many there are (more than LIST: no list).
    template <class F>
    SYN_DEV int gather(F&& pick) {
        if (threadIdx.x == 0) r.n = 0;
        __syncthreads();
        every([&](float v, int i) {
            if (!pick(v)) return;
            const uint32_t to = atomicAdd(&r.n, 1u);
            if (to < (uint32_t)LIST) r.keys[to] = sp_key(v, i);
        });
        __syncthreads();
        const int n = (int)r.n;
        if (n <= LIST) sort(n);
        return n;
    }
    // Up to 1024 keys: runs of 64 are put in order by counting the smaller ones in them, then each key's place is its
    // place in its run and the smaller ones of the other runs, by halving them (keys differ).  356 keys: 1.2 us; in
    // the general form below 8.2.
    SYN_DEV void sort(int n) {
        const int i = threadIdx.x, run0 = i & ~63;
        if (n <= ST) {
            const uint64_t k = i < n ? r.keys[i] : ~0ull;
            if (run0 < n) {
                if (i >= n) r.keys[i] = ~0ull;  // (behind the last one: as many as fill its run)
                wave_lds_sync();
                int c = 0;
                const ulonglong2* other = reinterpret_cast<const ulonglong2*>(r.keys + run0);
#pragma unroll 8
                for (int j = 0; j < 32; ++j) {
                    const ulonglong2 o = other[j];
                    c += (o.x < k ? 1 : 0) + (o.y < k ? 1 : 0);
                }
                wave_lds_sync();
                if (i < n) r.keys[run0 + c] = k;
            }
            __syncthreads();
            int place = 0;
            uint64_t mine = 0;
            if (run0 < n) {
                mine = r.keys[i];
                place = i & 63;
#pragma unroll 4
                for (int o = 0; o < n; o += 64) {
                    if (o == run0) continue;  // uniform
                    const int len = n - o < 64 ? n - o : 64;
                    int lo = 0;  // how many of it are smaller, a bit at a time
#pragma unroll
                    for (int d = 64; d >= 1; d /= 2) lo += lo + d <= len && r.keys[o + (lo + d <= len ? lo + d : 1) - 1] < mine ? d : 0;
                    place += lo;
                }
            }
            __syncthreads();
            if (i < n) r.keys[place] = mine;
            __syncthreads();
            return;
        }
        int size = 2 * ST;
        for (int p = n + threadIdx.x; p < size; p += ST) r.keys[p] = ~0ull;
        __syncthreads();
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                const int p = 2 * i - (i & (j - 1)), o = p + j;  // (bit j of p is 0)
                const uint64_t a = r.keys[p], b = r.keys[o];
                if ((a > b) == ((p & k) == 0)) r.keys[p] = b, r.keys[o] = a;
                __syncthreads();
            }
    }
    // The running sums of the list's n values: from `first` on for the first n0, from `second` on for the others.
    SYN_DEV void sum_list(int n, int n0, double first, double second) {
        static_assert(LIST == 2 * ST, "two keys a thread");
        double w[2], all;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * (int)threadIdx.x + j;
            w[j] = i < n ? sc.weight(sc.s(sp_of_key(r.keys[i]))) : 0.0;
        }
        const double s = before<double>(w[0] + w[1], r.part, all);
        r.run[2 * threadIdx.x] = s + w[0];
        r.run[2 * threadIdx.x + 1] = s + w[0] + w[1];
        __syncthreads();
        const double head = n0 > 0 && n0 < n ? r.run[n0 - 1] : 0.0;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * (int)threadIdx.x + j;
            r.run[i] = i < n0 ? first + r.run[i] : second + (r.run[i] - head);
        }
        __syncthreads();
    }
    // (every thread) The first of the list's values i0 .. i1 - 1 of which it is so; i1 where it is of none.
    template <class F>
    SYN_DEV int first(int i0, int i1, F&& so) {
        uint32_t v = 0xFFFFFFFFu;
#pragma unroll
        for (int j = 1; j >= 0; --j) {
            const int i = 2 * (int)threadIdx.x + j;
            if (i >= i0 && i < i1 && so(r.run[i], r.keys[i])) v = (uint32_t)i;
        }
        v = least(v);
        return v == 0xFFFFFFFFu ? i1 : (int)v;
    }

    // Where what is wanted is, in bin b: by the list of its values, or where they are too many for one digit by digit
    // of their keys.
    SYN_DEV Place find(Want want, uint32_t n, double sum) {
        if (threadIdx.x < 64) {
            const int o = bin_of(want, n, sum);
            if (threadIdx.x == 0) r.bin = o;
        }
        __syncthreads();
        const int b = r.bin;
        __syncthreads();
        if (r.in(b) <= (uint32_t)LIST) {
            const int m = gather([&](float v) { return v != -__builtin_inff() && Scale::bin(sc.s(v)) == b; });
            sum_list(m, m, r.base(b), 0.0);
            const uint32_t n0 = r.count0(b);
            const int at = want == AT_LEAST_N ? (int)(n - n0) - 1 : first(0, m, [&](double s, uint64_t) {
                return want == SUM_REACHES ? s >= sum : s > sum;
            });
            const int i = at < m ? at : m - 1;
            return Place{n0 + (uint32_t)i + 1, r.run[i], r.keys[i]};
        }
        return descend(b, want, n, sum);
    }
    SYN_DEV Place descend(int b, Want want, uint32_t n, double sum) {
        uint32_t* dcount = reinterpret_cast<uint32_t*>(r.run);  // [256]
        uint64_t* dmass = r.keys;
        const double unit = sc.unit(b);
        __syncthreads();
        if (threadIdx.x == 0) r.prefix = 0, r.before = r.count0(b), r.before_mass = 0;
#pragma unroll 1
        for (int shift = 56; shift >= 0; shift -= 8) {
            if (threadIdx.x < 256) dcount[threadIdx.x] = 0, dmass[threadIdx.x] = 0;
            __syncthreads();
            const uint64_t prefix = r.prefix;
            every([&](float v, int i) {
                if (v == -__builtin_inff()) return;
                const double s = sc.s(v);
                const uint64_t key = sp_key(v, i);
                if (Scale::bin(s) != b || (shift < 56 && (key >> (shift + 8)) != prefix)) return;
                atomicAdd(&dcount[key >> shift & 255], 1u);
                atomicAdd((unsigned long long*)&dmass[key >> shift & 255], (unsigned long long)sc.whole(s, b));
            });
            __syncthreads();
            if (threadIdx.x == 0) {
                int d = -1;
                uint32_t cn = r.before, at_n = cn;
                uint64_t ms = r.before_mass, at_ms = ms;
                for (int i = 0; i < 256; ++i) {
                    if (!dcount[i]) continue;
                    d = i, at_n = cn, at_ms = ms;
                    cn += dcount[i], ms += dmass[i];
                    const double c = r.base(b) + (double)ms * unit;
                    if (want == AT_LEAST_N ? cn >= n : want == SUM_REACHES ? c >= sum : c > sum) break;
                }
                r.prefix = r.prefix << 8 | (uint32_t)d;
                r.before = at_n, r.before_mass = at_ms;
                if (shift == 0) r.n = at_n + 1, r.sum = r.base(b) + (double)(at_ms + dmass[d]) * unit;
            }
            __syncthreads();
        }
        const Place p{r.n, r.sum, r.prefix};
        __syncthreads();
        return p;
    }

    // ---- the steps ------------------------------------------------------------------------------------------
    // (every thread gets it) the greatest of this workgroup's values, as sp_order
    SYN_DEV uint32_t greatest() {
        if (threadIdx.x == 0) r.most = 0;
        __syncthreads();
        uint32_t most = 0;
        each<true>([&](float v, int) {
            const uint32_t k = sp_order(v);
            most = k > most ? k : most;
        });
        most = group_max_u32<64>(most);
        if ((threadIdx.x & 63) == 0) atomicMax(&r.most, most);
        __syncthreads();
        return r.most;
    }
    SYN_DEV int bin32(float v) const {
        const float s = ((float)sc.m - v) * (float)sc.c;
        return s < (float)(SB - 1) ? (int)s : SB - 1;
    }
    // The counts (and sums) of the bins over this workgroup's values.
    SYN_DEV void bins(Mode mode) {
        for (int i = threadIdx.x; i < SLOTS; i += ST) r.counts[i] = 0, r.masses[i] = 0;
        __syncthreads();
        if (mode == LIST_K) {
            each<false>([&](float v, int) {
                if (v != -__builtin_inff()) atomicAdd(&r.counts[sp_at(bin32(v))], 1u);
            });
        } else {
            each<false>([&](float v, int) { add_to_bin(v); });
        }
        __syncthreads();
    }
    SYN_DEV void add_to_bin(float v) {
        if (v == -__builtin_inff()) return;
        const double s = sc.s(v);
        const int b = Scale::bin(s);
        atomicAdd(&r.counts[sp_at(b)], 1u);
        atomicAdd((unsigned long long*)&r.masses[sp_at(b)], (unsigned long long)sc.whole(s, b));
    }
    // (every thread gets it; behind a barrier) The bins before each, and from them what to gather, by one wavefront.
    SYN_DEV Wanted want(Mode mode) {
        if (mode == LIST_MIN_P) return Wanted{0, SB - 1, -1, -1, false, false, 0};
        if (threadIdx.x < 64) {
            const Wanted w = wanted(mode);
            if (threadIdx.x == 0) r.want = w;
        }
        __syncthreads();
        return r.want;
    }
    SYN_DEV Wanted wanted(Mode mode) {
        Wanted w{0, SB - 1, -1, -1, false, false, 0};
        prefix(mode == BINS);
        if (mode == LIST_K) {
            w.a1 = bin_of(AT_LEAST_N, q.k, 0.0);
            w.n = r.count0(w.a1 + 1);
            return w;
        }
        w.n = (uint32_t)LIST + 1;
        if (q.k < r.count0(SB)) return w;  // (a top-k longer than a list: its border, then the others', in seldom())
        const double all = r.base(SB);
        int p = SB, m = SB;
        if (q.top_p < 1.0f) p = bin_of(SUM_REACHES, 0, (double)q.top_p * all);
        if (q.min_p > 0.0f) m = Scale::bin(q.last);
        // (of two borders in different bins the first counts)
        if (p < SB || m < SB) {
            w.cut = p < m ? p : m;
            w.by_p = p == w.cut;
            w.by_min_p = m == w.cut;
        }
        // the token's sum lies between these, and its bin so
        const double lo = w.cut >= 0 ? r.base(w.cut) : all, hi = w.cut >= 0 ? r.base(w.cut + 1) : all;
        w.a0 = bin_of(SUM_PASSES, 0, (double)q.u * lo);
        w.a1 = w.cut >= 0 ? bin_of(SUM_PASSES, 0, (double)q.u * hi) : w.a0;
        if (w.a0 > w.a1) w.a0 = w.a1;
        if (w.cut >= 0) {
            if (w.cut <= w.a1 + 1)
                w.a1 = w.cut > w.a1 ? w.cut : w.a1;
            else
                w.b = w.cut;
        }
        w.n = r.count0(w.a1 + 1) - r.count0(w.a0) + (w.b >= 0 ? r.in(w.b) : 0);
        return w;
    }
    // The wanted among this workgroup's values: put(key) of each.
    template <class F>
    SYN_DEV void pick(Mode mode, const Wanted& w, F&& put) {
        if (mode == LIST_K) {
            each<false>([&](float v, int i) {
                if (v != -__builtin_inff() && bin32(v) <= w.a1) put(sp_key(v, i));
            });
        } else if (mode == LIST_MIN_P) {
            each<false>([&](float v, int i) {
                if (v != -__builtin_inff() && sc.s(v) <= q.last) put(sp_key(v, i));
            });
        } else {
            each<false>([&](float v, int i) {
                if (v == -__builtin_inff()) return;
                const int b = Scale::bin(sc.s(v));
                if ((b >= w.a0 && b <= w.a1) || b == w.b) put(sp_key(v, i));
            });
        }
    }
    SYN_DEV void write(const SampleArgs& g, uint64_t row, uint32_t kept, double w, uint64_t key) {
        if (threadIdx.x != 0) return;
        g.token[row] = (int)(uint32_t)key;
        g.kept[row] = (int)kept;
        const float lp = (float)(sc.s(sp_of_key(key)) * (-0.69314718055994530942 / 32.0) - log(w));
        g.logprob[row] = kept == 1 || lp > 0.0f ? 0.0f : lp;
    }
    static SYN_DEV void write_none(const SampleArgs& g, uint64_t row) {
        if (threadIdx.x == 0) g.token[row] = -1, g.logprob[row] = __builtin_nanf(""), g.kept[row] = 0;
    }
    // The row's results from the sorted list of the n wanted values; with more than LIST (no list) from the bins and the
    // row, all of which this workgroup then reads.
    SYN_DEV void finish(const SampleArgs& g, uint64_t row, Mode mode, const Wanted& w, uint32_t n) {
        if (n > (uint32_t)LIST) {
            seldom(g, row, mode);
            return;
        }
        // the list's border lies in its values i0 .. end - 1; `before` values stand before the i0th
        int n0 = (int)n, i0 = 0, end = q.k < n ? (int)q.k : (int)n;
        uint32_t before = 0;
        double base0 = 0.0, base1 = 0.0;
        if (mode == BINS) {
            n0 = (int)(r.count0(w.a1 + 1) - r.count0(w.a0)), end = (int)n;
            base0 = r.base(w.a0);
            if (w.b >= 0) base1 = r.base(w.b);
            if (w.cut >= 0) {
                i0 = w.b >= 0 ? n0 : (int)(r.count0(w.cut) - r.count0(w.a0));
                end = i0 + (int)r.in(w.cut);
                before = r.count0(w.cut);
            }
        }
        const bool cut = mode != BINS || w.cut >= 0, by_p = cut && q.top_p < 1.0f && (mode != BINS || w.by_p),
                   by_min_p = cut && q.min_p > 0.0f && (mode != BINS || w.by_min_p);
        auto results = [&](auto&& first_of, auto&& run, auto&& key) {
            if (by_p && end > i0) {
                const double reach = (double)q.top_p * (mode != BINS ? run(end - 1) : r.base(SB));
                const int at = first_of(i0, end, [&](double s, uint64_t) { return s >= reach; });
                end = at < end ? at + 1 : end;
            }
            if (by_min_p) end = first_of(i0, end, [&](double, uint64_t k) { return sc.s(sp_of_key(k)) > q.last; });
            const uint32_t kept = cut ? before + (uint32_t)(end - i0) : r.count0(SB);
            const double all = !cut ? r.base(SB) : end > i0 ? run(end - 1) : r.base(w.cut);
            // (where nothing of the cut's own bin is kept, the token lies in the first range)
            const double pass = (double)q.u * all;
            const int stop = end > 0 ? end : 1, at = first_of(0, stop, [&](double s, uint64_t) { return s > pass; });
            write(g, row, kept, all, key(at < stop ? at : stop - 1));
        };
        if (n <= 256) {  // by one wavefront, four neighbouring values a lane
            if (threadIdx.x >= 64) return;
            const int l = threadIdx.x;
            uint64_t k[4];
            double s[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int i = 4 * l + j;
                k[j] = i < (int)n ? r.keys[i] : 0;
                s[j] = i < (int)n ? sc.weight(sc.s(sp_of_key(k[j]))) : 0.0;
                if (j) s[j] += s[j - 1];
            }
            double up = s[3];
#pragma unroll
            for (int d = 1; d < 64; d *= 2) {
                const double o = __shfl_up(up, d);
                up += l >= d ? o : 0.0;
            }
            const double to = __shfl_up(up, 1), from = l ? to : 0.0;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] += from;
            auto of = [&](auto (&v)[4], int i) {  // (a uniform place)
                auto m = v[0];
#pragma unroll
                for (int j = 1; j < 4; ++j) m = (i & 3) == j ? v[j] : m;
                return __shfl(m, i >> 2);
            };
            const double head = n0 > 0 && n0 < (int)n ? of(s, n0 - 1) : 0.0;
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] = 4 * l + j < n0 ? base0 + s[j] : base1 + (s[j] - head);
            results(
                [&](int a, int b, auto&& so) {
                    int at = b;
#pragma unroll
                    for (int j = 3; j >= 0; --j) {
                        const uint64_t yes = __builtin_amdgcn_ballot_w64(4 * l + j >= a && 4 * l + j < b && so(s[j], k[j]));
                        const int f = yes ? 4 * (__builtin_ffsll((long long)yes) - 1) + j : b;
                        at = f < at ? f : at;
                    }
                    return at;
                },
                [&](int i) { return of(s, i); }, [&](int i) { return of(k, i); });
            return;
        }
        sum_list((int)n, n0, base0, base1);
        results([&](int a, int b, auto&& so) { return first(a, b, so); }, [&](int i) { return r.run[i]; }, [&](int i) { return r.keys[i]; });
    }
    // Border by border: the top-k's, the top-p's, min-p's, the token.
    SYN_DEV void seldom(const SampleArgs& g, uint64_t row, Mode mode) {
        if (mode != BINS) {
            for (int i = threadIdx.x; i < SLOTS; i += ST) r.counts[i] = 0, r.masses[i] = 0;
            __syncthreads();
            every([&](float v, int) { add_to_bin(v); });
            __syncthreads();
            if (threadIdx.x < 64) prefix(true);
            __syncthreads();
        }
        Place cut{r.count0(SB), r.base(SB), 0};
#pragma unroll 1
        for (int step = 0; step < 4; ++step) {
            Want want = AT_LEAST_N;
            uint32_t n = 0;
            double sum = 0.0;
            if (step == 0) {
                if (q.k >= cut.n) continue;
                n = q.k;
            } else if (step == 1) {
                if (q.top_p >= 1.0f) continue;
                want = SUM_REACHES, sum = (double)q.top_p * cut.sum;
            } else if (step == 2) {
                if (!(q.min_p > 0.0f)) continue;
                if (threadIdx.x == 0) r.n = 0;
                __syncthreads();
                uint32_t mine = 0;
                every([&](float v, int) { mine += v != -__builtin_inff() && sc.s(v) <= q.last ? 1 : 0; });
                atomicAdd(&r.n, mine);
                __syncthreads();
                n = r.n;
                __syncthreads();
                if (n >= cut.n) continue;
            } else {
                want = SUM_PASSES, sum = (double)q.u * cut.sum;
            }
            const Place p = find(want, n, sum);
            __syncthreads();
            if (step == 3)
                write(g, row, cut.n, cut.sum, p.key);
            else if (p.n < cut.n)
                cut = p;
        }
    }
};

}  // namespace

// ---- a row a workgroup --------------------------------------------------------------------------------------
template <int TY>
__global__ __launch_bounds__(ST) void k_sample(SampleArgs g) {
    const uint64_t row = blockIdx.x;
    __shared__ Row r;
    Sampler<TY> sp(g, row, r);
    if (!sp.set_most(sp.greatest())) {
        sp.write_none(g, row);
        return;
    }
    const Mode mode = sp.mode();
    if (mode != LIST_MIN_P) sp.bins(mode);
    const Wanted w = sp.want(mode);
    if (threadIdx.x == 0) r.n = 0;
    __syncthreads();
    if (w.n <= (uint32_t)LIST)
        sp.pick(mode, w, [&](uint64_t key) {
            const uint32_t to = atomicAdd(&r.n, 1u);
            if (to < (uint32_t)LIST) r.keys[to] = key;
        });
    __syncthreads();
    const uint32_t n = w.n <= (uint32_t)LIST ? r.n : w.n;
    __syncthreads();
    if (n <= (uint32_t)LIST) sp.sort((int)n);
    sp.finish(g, row, mode, w, n);
}

// ---- few long rows: a row's parts, a launch a step ------------------------------------------------------------
// A row's share of the workspace: the parts' greatest values, how many were gathered, the bins, the list.
struct Shared {
    uint32_t most[64];
    uint32_t n;
    uint32_t pad[63];
    uint32_t counts[SLOTS];
    uint64_t masses[SLOTS];
    uint64_t keys[LIST];
};
static_assert(SLOTS % 2 == 0, "the sums on 8 bytes");

template <int TY>
__global__ __launch_bounds__(ST) void k_sample_most(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    const int part = (int)(blockIdx.x % (uint32_t)parts);
    __shared__ Row r;
    Sampler<TY> sp(g, row, r);
    sp.take(part, parts);
    Shared& s = ((Shared*)g.ws)[row];
    for (int i = part * ST + (int)threadIdx.x; i < SLOTS; i += parts * ST) s.counts[i] = 0, s.masses[i] = 0;
    if (part == 0 && threadIdx.x == 0) s.n = 0;
    const uint32_t m = sp.greatest();
    if (threadIdx.x == 0) s.most[part] = m;
}
SYN_DEV uint32_t most_of(const Shared& s, int parts) {
    const int lane = threadIdx.x & 63;
    return group_max_u32<64>(lane < parts ? s.most[lane] : 0u);
}
template <int TY>
__global__ __launch_bounds__(ST) void k_sample_bins(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    __shared__ Row r;
    Sampler<TY> sp(g, row, r);
    sp.take((int)(blockIdx.x % (uint32_t)parts), parts);
    Shared& s = ((Shared*)g.ws)[row];
    if (!sp.set_most(most_of(s, parts)) || sp.mode() == LIST_MIN_P) return;
    const Mode mode = sp.mode();
    sp.bins(mode);
    for (int i = threadIdx.x; i < SLOTS; i += ST)  // (whole numbers: in any order)
        if (r.counts[i]) {
            atomicAdd(&s.counts[i], r.counts[i]);
            if (mode == BINS) atomicAdd((unsigned long long*)&s.masses[i], (unsigned long long)r.masses[i]);
        }
}
// The row's bins into LDS, and what to gather.
template <class S>
SYN_DEV Wanted want_shared(S& sp, const Shared& s, Row& r, Mode mode) {
    if (mode != LIST_MIN_P)
        for (int i = threadIdx.x; i < SLOTS; i += ST) r.counts[i] = s.counts[i], r.masses[i] = s.masses[i];
    __syncthreads();
    return sp.want(mode);
}
template <int TY>
__global__ __launch_bounds__(ST) void k_sample_pick(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    __shared__ Row r;
    Sampler<TY> sp(g, row, r);
    sp.take((int)(blockIdx.x % (uint32_t)parts), parts);
    Shared& s = ((Shared*)g.ws)[row];
    if (!sp.set_most(most_of(s, parts))) return;
    const Mode mode = sp.mode();
    const Wanted w = want_shared(sp, s, r, mode);
    if (w.n > (uint32_t)LIST) return;
    if (threadIdx.x == 0) r.n = 0;
    __syncthreads();
    sp.pick(mode, w, [&](uint64_t key) {
        const uint32_t to = atomicAdd(&r.n, 1u);
        if (to < (uint32_t)LIST) r.keys[to] = key;
    });
    __syncthreads();
    // (a place for all of this workgroup's at once: one by one, 24 rows' lists took 15 us)
    if (threadIdx.x == 0) r.at = r.n ? atomicAdd(&s.n, r.n) : 0;
    __syncthreads();
    const uint32_t n = r.n, at = r.at;
    for (uint32_t i = threadIdx.x; i < n && i < (uint32_t)LIST; i += ST)
        if (at + i < (uint32_t)LIST) s.keys[at + i] = r.keys[i];
}
template <int TY>
__global__ __launch_bounds__(ST) void k_sample_end(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x;
    __shared__ Row r;
    Sampler<TY> sp(g, row, r);
    Shared& s = ((Shared*)g.ws)[row];
    if (!sp.set_most(most_of(s, parts))) {
        sp.write_none(g, row);
        return;
    }
    const Mode mode = sp.mode();
    const Wanted w = want_shared(sp, s, r, mode);
    const uint32_t n = w.n <= (uint32_t)LIST ? s.n : w.n;
    if (n <= (uint32_t)LIST) {
        for (int i = threadIdx.x; i < (int)n; i += ST) r.keys[i] = s.keys[i];
        __syncthreads();
        sp.sort((int)n);
    }
    sp.finish(g, row, mode, w, n);
}

// How many workgroups share a row: as many as fill the chip twice, of 8192 values at least.
static int sample_parts(int xtype, int rows, int vocab) {
    if (rows > 128 || vocab <= (xtype == T_F32 ? 32768 : 65536)) return 1;
    const int most = vocab / 8192 < 64 ? vocab / 8192 : 64, parts = 512 / rows;
    return parts < most ? parts : most;
}

uint64_t sample_ws_bytes(int xtype, int rows, int vocab) {
    return sample_parts(xtype, rows, vocab) > 1 ? align_up((uint64_t)rows * sizeof(Shared), 256) : 0;
}

template <int TY>
static void sample_as(const SampleArgs& a, hipStream_t stream) {
    const int parts = sample_parts(a.xtype, a.rows, a.vocab);
    if (parts > 1) {
        const dim3 all((uint32_t)a.rows * (uint32_t)parts);
        hipLaunchKernelGGL(k_sample_most<TY>, all, dim3(ST), 0, stream, a, parts);
        hipLaunchKernelGGL(k_sample_bins<TY>, all, dim3(ST), 0, stream, a, parts);
        hipLaunchKernelGGL(k_sample_pick<TY>, all, dim3(ST), 0, stream, a, parts);
        hipLaunchKernelGGL(k_sample_end<TY>, dim3(a.rows), dim3(ST), 0, stream, a, parts);
    } else {
        hipLaunchKernelGGL(k_sample<TY>, dim3(a.rows), dim3(ST), 0, stream, a);
    }
}

void launch_sample(const SampleArgs& a, hipStream_t stream) {
    if (a.xtype == T_F32)
        sample_as<T_F32>(a, stream);
    else if (a.xtype == T_F16)
        sample_as<T_F16>(a, stream);
    else
        sample_as<T_BF16>(a, stream);
}

}  // namespace syn
