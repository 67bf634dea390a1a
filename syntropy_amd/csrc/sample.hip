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

// The scale of a row's distances and of its weights.
struct Scale {
    double m, c;  // the greatest logit; 32 log2(e) / T
    double one;   // 2^bits: the whole number of a bin's middle weight
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
    SYN_DEV double unit(int b) const { return exp2((double)b * (-1.0 / 32.0)) / one; }
};

enum Want { AT_LEAST_N, SUM_REACHES, SUM_PASSES };

constexpr int LIST = 2048;  // keys that a workgroup sorts

struct Row {
    uint32_t count0[SB + 1];  // of a bin's values, then of those before it
    uint64_t mass[SB + 1];    // of a bin, then (as double) the sum before it
    uint64_t keys[LIST];      // the gathered values' keys: (order from above, index), so that they order upwards
    double run[LIST];         // the running sum at each, from the row's first value on
    double part[ST / 64];
    uint32_t npart[ST / 64];
    uint32_t most, at, n;
    // of descend()
    uint64_t prefix, before_mass;
    uint32_t before;
    double sum;
    SYN_DEV double base(int b) const { return __builtin_bit_cast(double, mass[b]); }
    SYN_DEV uint32_t in(int b) const { return count0[b + 1] - count0[b]; }
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
    const uint8_t* x;
    int vocab;
    Scale sc;
    Row& r;

    // f(value, index) of every value, 16 bytes a load, at any value's address
    template <class F>
    SYN_DEV void each(F&& f) const {
        constexpr int PER = TY == T_F32 ? 4 : 8, MANY = 4, ES = TY == T_F32 ? 4 : 2;
        const int whole = vocab / PER;
        for (int p = threadIdx.x; p < whole; p += ST * MANY) {
            uint32_t w[MANY][4];
#pragma unroll
            for (int m = 0; m < MANY; ++m) {
                const int q = p + ST * m < whole ? p + ST * m : p;
                __builtin_memcpy(w[m], x + (int64_t)q * (PER * ES), 16);
            }
#pragma unroll
            for (int m = 0; m < MANY; ++m) {
                if (p + ST * m >= whole) break;
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    float v;
                    if constexpr (TY == T_F32) {
                        v = u2f(w[m][j]);
                    } else {
                        const uint32_t h = w[m][j / 2];
                        v = TY == T_F16 ? f16_to_f32(j & 1 ? h >> 16 : h) : u2f(j & 1 ? h & 0xFFFF0000u : h << 16);
                    }
                    f(v, (p + ST * m) * PER + j);
                }
            }
        }
        const int i = whole * PER + (int)threadIdx.x;
        if (i < vocab) f(sp_load<TY>(x, i), i);
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

    // Counts, then also sums, of the bins before each, in place.
    SYN_DEV void prefix_counts() {
        static_assert(SB == 2 * ST, "two bins a thread");
        uint32_t c[2], all;
        c[0] = r.count0[2 * threadIdx.x], c[1] = r.count0[2 * threadIdx.x + 1];
        const uint32_t b = before<uint32_t>(c[0] + c[1], r.npart, all);
        r.count0[2 * threadIdx.x] = b;
        r.count0[2 * threadIdx.x + 1] = b + c[0];
        if (threadIdx.x == 0) r.count0[SB] = all;
        __syncthreads();
    }
    SYN_DEV void prefix_sums() {
        double m[2], all;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int b = 2 * (int)threadIdx.x + j;
            m[j] = r.mass[b] ? (double)r.mass[b] * sc.unit(b) : 0.0;
        }
        const double s = before<double>(m[0] + m[1], r.part, all);
        r.mass[2 * threadIdx.x] = __builtin_bit_cast(uint64_t, s);
        r.mass[2 * threadIdx.x + 1] = __builtin_bit_cast(uint64_t, s + m[0]);
        if (threadIdx.x == 0) r.mass[SB] = __builtin_bit_cast(uint64_t, all);
        __syncthreads();
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
    // The first bin whose values reach what is wanted (the last that holds any where none does).
    SYN_DEV int bin_of(Want want, uint32_t n, double sum) {
        uint32_t b = 0xFFFFFFFFu, held = 0xFFFFFFFFu;
#pragma unroll
        for (int j = 1; j >= 0; --j) {
            const int i = 2 * (int)threadIdx.x + j;
            if (!r.in(i)) continue;
            if (held == 0xFFFFFFFFu) held = (uint32_t)(SB - 1 - i);
            const bool yes = want == AT_LEAST_N ? r.count0[i + 1] >= n : want == SUM_REACHES ? r.base(i + 1) >= sum : r.base(i + 1) > sum;
            if (yes) b = (uint32_t)i;
        }
        b = least(b);
        if (b == 0xFFFFFFFFu) b = (uint32_t)(SB - 1) - least(held);
        return (int)b;
    }

    // The keys that `pick` takes, in order, into r.keys; returns how many there are (more than LIST: no list).
    template <class F>
    SYN_DEV int gather(F&& pick) {
        if (threadIdx.x == 0) r.n = 0;
        __syncthreads();
        each([&](float v, int i) {
            if (!pick(v)) return;
            const uint32_t to = atomicAdd(&r.n, 1u);
            if (to < (uint32_t)LIST) r.keys[to] = sp_key(v, i);
        });
        __syncthreads();
        const int n = (int)r.n;
        if (n <= LIST) sort(n);
        return n;
    }
    SYN_DEV void sort(int n) {
        if (n <= 256) {  // each finds its place by counting the smaller ones: four wavefronts' keys, a quarter each
            uint32_t* rank = reinterpret_cast<uint32_t*>(r.run);
            const int i = threadIdx.x & 255, q = threadIdx.x >> 8;
            if (threadIdx.x < 256) rank[threadIdx.x] = 0;
            __syncthreads();
            const uint64_t k = i < n ? r.keys[i] : 0;
            uint32_t c = 0;
            for (int j = q * n / 4; j < (q + 1) * n / 4; ++j) c += r.keys[j] < k ? 1 : 0;
            if (i < n && c) atomicAdd(&rank[i], c);
            __syncthreads();
            if (q == 0 && i < n) r.keys[rank[i]] = k;
            __syncthreads();
            return;
        }
        int size = 512;
        while (size < n) size *= 2;
        for (int i = n + threadIdx.x; i < size; i += ST) r.keys[i] = ~0ull;
        __syncthreads();
        for (int k = 2; k <= size; k *= 2)
            for (int j = k / 2; j > 0; j /= 2) {
                for (int p = threadIdx.x; p < size / 2; p += ST) {
                    const int i = 2 * p - (p & (j - 1)), o = i + j;  // (bit j of i is 0)
                    const uint64_t a = r.keys[i], b = r.keys[o];
                    if ((a > b) == ((i & k) == 0)) r.keys[i] = b, r.keys[o] = a;
                }
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
    // The first of the list's values i0 .. i1 - 1 of which it is so, or the last of them.
    template <class F>
    SYN_DEV int first(int i0, int i1, F&& so) {
        uint32_t v = 0xFFFFFFFFu;
#pragma unroll
        for (int j = 1; j >= 0; --j) {
            const int i = 2 * (int)threadIdx.x + j;
            if (i >= i0 && i < i1 && so(i)) v = (uint32_t)i;
        }
        v = least(v);
        return v == 0xFFFFFFFFu ? i1 - 1 : (int)v;
    }

    // Where what is wanted is, in bin b: by the list of its values, or where they are too many for one digit by digit
    // of their keys.
    SYN_DEV Place find(Want want, uint32_t n, double sum) {
        const int b = bin_of(want, n, sum);
        if (r.in(b) <= (uint32_t)LIST) {
            const int m = gather([&](float v) { return v != -__builtin_inff() && Scale::bin(sc.s(v)) == b; });
            sum_list(m, m, r.base(b), 0.0);
            return place(first(0, m, [&](int i) {
                return want == AT_LEAST_N ? r.count0[b] + i + 1 >= n : want == SUM_REACHES ? r.run[i] >= sum : r.run[i] > sum;
            }), r.count0[b]);
        }
        return descend(b, want, n, sum);
    }
    SYN_DEV Place place(int i, uint32_t before) const { return Place{before + (uint32_t)i + 1, r.run[i], r.keys[i]}; }

    SYN_DEV Place descend(int b, Want want, uint32_t n, double sum) {
        uint32_t* dcount = reinterpret_cast<uint32_t*>(r.run);  // [256]
        uint64_t* dmass = r.keys;
        const double unit = sc.unit(b);
        __syncthreads();
        if (threadIdx.x == 0) r.prefix = 0, r.before = r.count0[b], r.before_mass = 0;
#pragma unroll 1
        for (int shift = 56; shift >= 0; shift -= 8) {
            if (threadIdx.x < 256) dcount[threadIdx.x] = 0, dmass[threadIdx.x] = 0;
            __syncthreads();
            const uint64_t prefix = r.prefix;
            each([&](float v, int i) {
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
};

}  // namespace

template <int TY>
__global__ __launch_bounds__(ST) void k_sample(SampleArgs g) {
    const uint64_t row = blockIdx.x;
    __shared__ Row r;
    const float temperature = g.temperature ? g.temperature[row] : g.temperature0;
    const int top_k = g.top_k ? g.top_k[row] : g.top_k0;
    const float top_p = g.top_p ? g.top_p[row] : g.top_p0;
    float min_p = g.min_p ? g.min_p[row] : g.min_p0;
    float u = g.u[row];
    const bool greedy = temperature == 0.0f;
    Sampler<TY> sp{(const uint8_t*)g.x + row * g.ldx * (TY == T_F32 ? 4 : 2), g.vocab, {}, r};
    if (threadIdx.x == 0) r.most = 0;
    __syncthreads();
    uint32_t most = 0;
    sp.each([&](float v, int) {
        const uint32_t k = sp_order(v);
        most = k > most ? k : most;
    });
    most = group_max_u32<64>(most);
    if ((threadIdx.x & 63) == 0) atomicMax(&r.most, most);
    __syncthreads();
    most = r.most;
    const bool fit = greedy || (temperature >= 0x1p-64f && temperature <= 0x1p64f);
    if (most >= KEY_INF || most <= KEY_NONE || !fit || top_p != top_p || min_p != min_p || u != u) {
        if (threadIdx.x == 0) g.token[row] = -1, g.logprob[row] = __builtin_nanf(""), g.kept[row] = 0;
        return;
    }
    int bits = 62;
    for (uint32_t v = 1; v < (uint32_t)g.vocab; v *= 2) --bits;
    Scale& sc = sp.sc;
    sc.m = sp_value(most);
    sc.c = 32.0 * 1.44269504088896340736 / (greedy ? 1.0 : (double)temperature);
    sc.one = ldexp(1.0, bits < 50 ? bits : 50);
    min_p = min_p < 1.0f ? min_p : 1.0f;
    const double last = min_p > 0.0f ? -32.0 * log2((double)min_p) : __builtin_inf();  // the greatest s that min-p keeps
    u = u < 0.0f ? 0.0f : u > 0x1.fffffep-1f ? 0x1.fffffep-1f : u;
    const uint32_t k = greedy ? 1u : top_k > 0 ? (uint32_t)top_k : 0xFFFFFFFFu;

    // The row's first values, as many as can count, as one list.
    auto finish = [&](uint32_t kept, double w, uint64_t key) {
        if (threadIdx.x != 0) return;
        const int id = (int)(uint32_t)key;
        g.token[row] = id;
        g.kept[row] = (int)kept;
        const float lp = (float)(sc.s(sp_of_key(key)) * (-0.69314718055994530942 / 32.0) - log(w));
        g.logprob[row] = kept == 1 || lp > 0.0f ? 0.0f : lp;
    };
    int m = LIST + 1;
    if (k <= (uint32_t)LIST && k < (uint32_t)g.vocab) {
        // top-k: the bins of as many values, by F32 distances (a count needs no weights)
        const float mf = sp_value(most), cf = (float)sc.c;
        auto bin = [&](float v) {
            const float s = (mf - v) * cf;
            return s < (float)(SB - 1) ? (int)s : SB - 1;
        };
        for (int i = threadIdx.x; i < SB; i += ST) r.count0[i] = 0;
        __syncthreads();
        sp.each([&](float v, int) {
            if (v != -__builtin_inff()) atomicAdd(&r.count0[bin(v)], 1u);
        });
        __syncthreads();
        sp.prefix_counts();
        const int b = sp.bin_of(AT_LEAST_N, k, 0.0);
        if (r.count0[b + 1] <= (uint32_t)LIST) m = sp.gather([&](float v) { return v != -__builtin_inff() && bin(v) <= b; });
        __syncthreads();
    } else if (top_p >= 1.0f && min_p > 0.0f) {
        m = sp.gather([&](float v) { return v != -__builtin_inff() && sc.s(v) <= last; });
        __syncthreads();
    }
    if (m <= LIST) {
        int n = k < (uint32_t)m ? (int)k : m;
        sp.sum_list(m, m, 0.0, 0.0);
        if (top_p < 1.0f) {
            const double reach = (double)top_p * r.run[n - 1];
            n = sp.first(0, n, [&](int i) { return r.run[i] >= reach; }) + 1;
        }
        if (min_p > 0.0f) {
            const int out = sp.first(0, n, [&](int i) { return sc.s(sp_of_key(r.keys[i])) > last; });
            n = out < n && sc.s(sp_of_key(r.keys[out])) > last ? out : n;
        }
        const double w = r.run[n - 1], pass = (double)u * w;
        finish((uint32_t)n, w, r.keys[sp.first(0, n, [&](int i) { return r.run[i] > pass; })]);
        return;
    }

    // The bins' counts and sums.
    for (int i = threadIdx.x; i < SB; i += ST) r.count0[i] = 0, r.mass[i] = 0;
    __syncthreads();
    sp.each([&](float v, int) {
        if (v == -__builtin_inff()) return;
        const double s = sc.s(v);
        const int b = Scale::bin(s);
        atomicAdd(&r.count0[b], 1u);
        atomicAdd((unsigned long long*)&r.mass[b], (unsigned long long)sc.whole(s, b));
    });
    __syncthreads();
    sp.prefix_counts();
    sp.prefix_sums();
    Place cut{r.count0[SB], r.base(SB), 0};
    if (k < cut.n) cut = sp.find(AT_LEAST_N, k, 0.0);
    if (top_p < 1.0f) {
        const Place p = sp.find(SUM_REACHES, 0, (double)top_p * cut.sum);
        if (p.n < cut.n) cut = p;
    }
    if (min_p > 0.0f) {
        if (threadIdx.x == 0) r.n = 0;
        __syncthreads();
        uint32_t mine = 0;
        sp.each([&](float v, int) { mine += v != -__builtin_inff() && sc.s(v) <= last ? 1 : 0; });
        atomicAdd(&r.n, mine);
        __syncthreads();
        const uint32_t reach = r.n;
        __syncthreads();
        if (reach < cut.n) cut = sp.find(AT_LEAST_N, reach, 0.0);
    }
    finish(cut.n, cut.sum, sp.find(SUM_PASSES, 0, (double)u * cut.sum).key);
}

uint64_t sample_ws_bytes(int, int) { return 0; }

void launch_sample(const SampleArgs& a, hipStream_t stream) {
    if (a.xtype == T_F32)
        hipLaunchKernelGGL(k_sample<T_F32>, dim3(a.rows), dim3(ST), 0, stream, a);
    else if (a.xtype == T_F16)
        hipLaunchKernelGGL(k_sample<T_F16>, dim3(a.rows), dim3(ST), 0, stream, a);
    else
        hipLaunchKernelGGL(k_sample<T_BF16>, dim3(a.rows), dim3(ST), 0, stream, a);
}

}  // namespace syn
