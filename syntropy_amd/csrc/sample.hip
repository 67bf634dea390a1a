// A token of each row of logits x [rows][vocab] by temperature T, top-k, top-p, min-p and a given u in [0, 1).
// The row's logits in order (descending, the lower index first among equals), w_i = exp((x_i - max x) / T):
//   top-k keeps the first k; top-p the least n of those whose sum of w reaches p times theirs; min-p those with
//   w_i >= min_p.  Each keeps a first part of the order, so all together do: n values, of the sum W.
//   The token is the first of them whose running sum passes u W.
// T = 0 stands for top-k 1.
//
// A token and a count are whole numbers, and the borders between tokens are as near to one another as 1e-6 of W, so
// sums have to be exact to far less than that, and the same whatever their order: with t_i = (max x - x_i) log2(e) / T in
// 64 bits, values are put in bins of 1/32 of t, and a bin's weights are added as whole numbers of 2^-bits of the weight in
// the bin's middle.  A bin is a run of the order; a prefix of the order is whole bins, whose sums are whole numbers
// too, of 2^-bits of the greatest weight, and a part of one, whose values are put in order as a list.
// A weight is off by 2^-48 of itself (the exponential's polynomial) and half of its whole number's 1, equal logits all the
// same way; a bin's sum by half of 2^-bits of the greatest weight, which is 2^(10 - bits) over all bins and the most of it.
// bits is min(50, 62 - log2 vocab rounded up), 45 at 128256 logits: together below 2^(11 - bits) of the row's sum.
//
// The row is read for its greatest value, for the bins, and for the list: the few values that a border or the token can
// lie among.  A top-k needs no bins: up to TOP the k-th of the 256 groups' greatest values is a bound that only a few
// values more than k reach, a longer one takes counts of F32 distances; with min-p alone the border is a value.  In a flat
// row the bins of border and token may hold more than a list: then they take one after the other (`only`).  More of a bin
// than a list holds (a high temperature, equal values by the thousand), or a longer top-k: each border is found digit
// by digit of the values' keys.
// What bounds it is the arithmetic of a workgroup's passes (a CU takes 1024 threads' instruction in 16 cycles: 20
// instructions a value are 0.08 us a 1024 values) and its steps between them; few long rows are therefore split over
// workgroups, a launch a step.
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace syn {

namespace {

constexpr int SB = 2048;        // bins; the last one holds all that is below 2^-64 too (as nothing)
constexpr int ST = 1024;        // threads a workgroup
constexpr int LIST = 64 * 31;   // values of a list: an odd number a lane, so that lanes' runs lie in different banks
constexpr uint32_t TOP = 64;
constexpr uint32_t KEY_INF = 0xFF800000u, KEY_NONE = 0x007FFFFFu;  // sp_order of +-infinity

// A whole number that orders as the value does (-0 as +0, every NaN above +infinity).
SYN_DEV uint32_t sp_order(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = f2u(v + 0.0f);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
SYN_DEV float sp_value(uint32_t k) { return u2f(k >> 31 ? k ^ 0x80000000u : ~k); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template <int TY>
SYN_DEV float sp_load(const uint8_t* row, int64_t i) {
    if constexpr (TY == T_F32) return ((const float*)row)[i];
    const uint32_t h = ((const uint16_t*)row)[i];
    return TY == T_F16 ? f16_to_f32(h) : u2f(h << 16);
}

// A value's key: (order from above, index), so that keys order upwards.
SYN_DEV uint64_t sp_key(float v, int i) { return (uint64_t)~sp_order(v) << 32 | (uint32_t)i; }
SYN_DEV float sp_of_key(uint64_t k) { return sp_value(~(uint32_t)(k >> 32)); }

// 2^(-j / 32)
__constant__ const double STEPS[32] = {
    0x1.0000000000000p+0, 0x1.f50765b6e4540p-1, 0x1.ea4afa2a490dap-1, 0x1.dfc97337b9b5fp-1, 0x1.d5818dcfba487p-1,
    0x1.cb720dcef9069p-1, 0x1.c199bdd85529cp-1, 0x1.b7f76f2fb5e47p-1, 0x1.ae89f995ad3adp-1, 0x1.a5503b23e255dp-1,
    0x1.9c49182a3f090p-1, 0x1.93737b0cdc5e5p-1, 0x1.8ace5422aa0dbp-1, 0x1.82589994cce13p-1, 0x1.7a11473eb0187p-1,
    0x1.71f75e8ec5f74p-1, 0x1.6a09e667f3bcdp-1, 0x1.6247eb03a5585p-1, 0x1.5ab07dd485429p-1, 0x1.5342b569d4f82p-1,
    0x1.4bfdad5362a27p-1, 0x1.44e086061892dp-1, 0x1.3dea64c123422p-1, 0x1.371a7373aa9cbp-1, 0x1.306fe0a31b715p-1,
    0x1.29e9df51fdee1p-1, 0x1.2387a6e756238p-1, 0x1.1d4873168b9aap-1, 0x1.172b83c7d517bp-1, 0x1.11301d0125b51p-1,
    0x1.0b5586cf9890fp-1, 0x1.059b0d3158574p-1};

// L^n / n!, n = 1 .. 5, of L = -ln 2 / 32: read to scalar registers, for as literals each would be moved to vector ones
// before its use.
__constant__ const double EXPS[5] = {-0x1.62e42fefa39efp-6, 0x1.ebfbdff82c58fp-13, -0x1.c6b08d704a0c0p-20, 0x1.3b2ab6fba4e77p-27, -0x1.5d87fe78a6731p-35};

// The scale of a row's distances and of its weights.
struct Scale {
    double m, c;  // the greatest logit; 32 log2(e) / T
    double one;   // 2^bits: the whole number of a bin's middle weight
    int bits;
    // 32 t of a value
    SYN_DEV double s(float x) const { return (m - (double)x) * c; }
    // a bin, and the weight of s as a whole number in it: 2^(-(s - bin) / 32), |s - bin| <= 1/2 (and where s is 0 exactly 1,
    // so that equal logits have borders where they are to have them); what is below 2^-64 as that
    struct Part {
        int bin;
        uint64_t whole;
    };
    static SYN_DEV int bin(double s) { return (int)__builtin_rint(__builtin_fmin(s, (double)(SB - 1))); }
    SYN_DEV Part part(double s) const { return inside(__builtin_fmin(s, (double)(SB - 1))); }
    SYN_DEV Part inside(double s) const {
        const double n = __builtin_rint(s), y = s - n;
        // exp(L y) one, whose 1 one is added with 2^52: the sum's last bits are the whole number
        double p = __builtin_fma(y, EXPS[4], EXPS[3]);
        p = __builtin_fma(p, y, EXPS[2]);
        p = __builtin_fma(p, y, EXPS[1]);
        p = __builtin_fma(p, y, EXPS[0]);
        return {(int)n, __builtin_bit_cast(uint64_t, __builtin_fma(p * one, y, one + 0x1p52)) & 0xFFFFFFFFFFFFFull};
    }
    SYN_DEV double weight(double s) const { return exp2(s * (-1.0 / 32.0)); }
    // what a whole number of bin b stands for, in 2^-bits of the greatest weight
    static SYN_DEV double step(int b) { return ldexp(STEPS[b & 31], -(b >> 5)); }
};

enum Want { AT_LEAST_N, SUM_REACHES, SUM_PASSES };
// How a row's list is found: a short top-k by a bound, a longer one by counts, min-p alone, the bins' sums.
enum Mode { LIST_TOP, LIST_K, LIST_MIN_P, BINS };

// What is gathered: of LIST_TOP the values from a bound on, of LIST_K the F32 bins up to a1, of LIST_MIN_P what min-p
// keeps, of BINS those from a0 to a1 and b.
struct Wanted {
    int a0, a1, b;   // (b: none where negative)
    int cut;         // BINS: the bin of the border (none: -1)
    bool by_p, by_min_p;
    bool only;       // BINS: only the border's bin, for the list holds not all; the token's after it
    uint32_t n;      // how many values that is (0: not known), or more than LIST: no list
    float lo, hi, lo2, hi2;  // the values from lo to below hi and from lo2 to below hi2
    // The list: its first n0 values are a0's to a1's, which `sum0` stands before, the others b's, which `sum1` does; the
    // border lies in its places i0 .. end - 1, which `before` values of the sum `under` stand before.  The row's own.
    int n0, i0, end;
    uint32_t before, total;
    double sum0, sum1, under, all;
    double to;  // of the other modes: about how far its last value lies
};

// A place in the order: how many values reach it, their sum, and the key of the last one.
struct Place {
    uint32_t n;
    double sum;
    uint64_t key;
};

struct Row {
    uint32_t counts[SB + 1];              // of a bin's values, then of those before it
    uint64_t masses[SB + 1];              // of a bin, then of those before it
    alignas(16) uint64_t keys[2 * ST];    // the gathered values' keys
    double run[2 * ST];                   // their weights, then the running sums
    uint32_t buckets[ST + 1], ends[5];    // of order()
    uint32_t part_n[ST / 64];
    uint64_t part_s[ST / 64];
    uint32_t most, n, at;
    int bin;
    Wanted want;
    Place place;
    // of digits()
    uint64_t prefix, before_mass;
    uint32_t before;
    SYN_DEV uint32_t in(int b) const { return counts[b + 1] - counts[b]; }
};

// A row's values, or a workgroup's part of them.
template <int TY>
struct Reader {
    static constexpr int PER = TY == T_F32 ? 4 : 8, ES = TY == T_F32 ? 4 : 2;
    const uint8_t* x;
    int vocab;
    int first_piece, end_piece;  // of 16 bytes (the row's last values are the last part's)

    SYN_DEV Reader(const SampleArgs& g, uint64_t row, int part, int parts) : x((const uint8_t*)g.x + row * g.ldx * ES), vocab(g.vocab) {
        const int all = vocab / PER;
        first_piece = (int)((int64_t)all * part / parts);
        end_piece = (int)((int64_t)all * (part + 1) / parts);
    }
    SYN_DEV static float value(u32x4 w, int j) {
        if constexpr (TY == T_F32) return u2f(w[j]);
        const uint32_t h = w[j / 2];
        if constexpr (TY == T_F16) return f16_to_f32(j & 1 ? h >> 16 : h);
        return u2f(j & 1 ? h & 0xFFFF0000u : h << 16);
    }
    // f(16 bytes, the index of their first value) of this workgroup's, at any value's address; then rest(value, index) of
    // the row's last ones.  Four loads are in flight, passed down (moves) to one copy of f: code that is run once
    // costs its way into the instruction cache (with four copies, and the steps below as often as they are used, a
    // row of 32064 took 3 us more).
    template <class F, class G>
    SYN_DEV void pieces(F&& f, G&& rest) const {
        constexpr int MANY = 4;
        u32x4 w[MANY];
        auto load = [&](int p) {
            u32x4 v;
            __builtin_memcpy(&v, x + (int64_t)(p < end_piece ? p : first_piece) * 16, 16);
            return v;
        };
        if (first_piece < end_piece) {
            int p = first_piece + (int)threadIdx.x;
#pragma unroll
            for (int m = 0; m < MANY; ++m) w[m] = load(p + ST * m);
#pragma unroll 1
            for (; p < end_piece; p += ST) {
                const u32x4 o = w[0];
#pragma unroll
                for (int m = 0; m + 1 < MANY; ++m) w[m] = w[m + 1];
                w[MANY - 1] = load(p + ST * MANY);
                f(o, p * PER);
            }
        }
        const int i = vocab / PER * PER + (int)threadIdx.x;
        if (i < vocab && end_piece == vocab / PER) rest(sp_load<TY>(x, i), i);
    }
    template <class F>
    SYN_DEV void each(F&& f) const {
        pieces([&](u32x4 w, int i) {
#pragma unroll
            for (int j = 0; j < PER; ++j) f(value(w, j), i + j);
        }, f);
    }
    // The same of the whole row, value by value: for what is seldom.
    template <class F>
    SYN_DEV void every(F&& f) const {
#pragma unroll 1
        for (int i = threadIdx.x; i < vocab; i += ST) f(sp_load<TY>(x, i), i);
    }

    // ---- the greatest value ---------------------------------------------------------------------------------
    // sp_order of the greatest of this thread's values, from the greatest as signed and unsigned words and the least as
    // unsigned ones (of 16 bits two at a time): the first is it unless all are negative, then the last is; and a
    // NaN shows in one of the first two.
    SYN_DEV uint32_t greatest() const {
        if constexpr (TY == T_F32) {
            uint32_t us = 0xFF800000u, ul = us;
            int32_t sg = (int32_t)us;
            auto add = [&](uint32_t b) {
                sg = (int32_t)b > sg ? (int32_t)b : sg;
                us = b > us ? b : us;
                ul = b < ul ? b : ul;
            };
            pieces([&](u32x4 w, int) {
#pragma unroll
                for (int j = 0; j < 4; ++j) add(w[j]);
            }, [&](float v, int) { add(f2u(v)); });
            if (sg > 0x7F800000 || us > 0xFF800000u) return 0xFFFFFFFFu;
            return sp_order(u2f(sg >= 0 ? (uint32_t)sg : ul));
        } else {
            typedef short s16x2 __attribute__((ext_vector_type(2)));
            typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
            constexpr uint16_t INF = TY == T_F16 ? 0x7C00 : 0x7F80, NONE = INF | 0x8000;
            s16x2 sg = {(short)NONE, (short)NONE};
            u16x2 us = {NONE, NONE}, ul = us;
            auto add = [&](uint32_t b) {
                const s16x2 s = __builtin_bit_cast(s16x2, b);
                const u16x2 v = __builtin_bit_cast(u16x2, b);
                sg = __builtin_elementwise_max(sg, s);
                us = __builtin_elementwise_max(us, v);
                ul = __builtin_elementwise_min(ul, v);
            };
            uint32_t more = 0;
            pieces([&](u32x4 w, int) {
#pragma unroll
                for (int j = 0; j < 4; ++j) add(w[j]);
            }, [&](float v, int) { more = sp_order(v); });
            const short s = sg[0] > sg[1] ? sg[0] : sg[1];
            const uint16_t m = us[0] > us[1] ? us[0] : us[1], l = ul[0] < ul[1] ? ul[0] : ul[1];
            uint32_t k = 0xFFFFFFFFu;
            if (s <= (short)INF && m <= NONE) {
                const uint32_t b = s >= 0 ? (uint32_t)(uint16_t)s : l;
                k = sp_order(TY == T_F16 ? f16_to_f32(b) : u2f(b << 16));
            }
            return k > more ? k : more;
        }
    }
};

template <int TY>
struct Sampler : Reader<TY> {
    using Reader<TY>::vocab, Reader<TY>::each, Reader<TY>::every;
    Row& r;
    // the row's settings
    float temperature, top_p, min_p, u;
    int top_k;
    // what follows from them and the greatest value
    Scale sc;
    uint32_t k;      // (all: 2^32 - 1)
    double last;     // the greatest s that min-p keeps

    SYN_DEV Sampler(const SampleArgs& g, uint64_t row, Row& rr, int part = 0, int parts = 1) : Reader<TY>(g, row, part, parts), r(rr) {
        temperature = g.temperature ? g.temperature[row] : g.temperature0;
        top_k = g.top_k ? g.top_k[row] : g.top_k0;
        top_p = g.top_p ? g.top_p[row] : g.top_p0;
        min_p = g.min_p ? g.min_p[row] : g.min_p0;
        u = g.u[row];
    }
    // false: the row has no distribution, or its settings say nothing
    SYN_DEV bool settle(uint32_t most) {
        const bool greedy = temperature == 0.0f;
        if (!(greedy || (temperature >= 0x1p-64f && temperature <= 0x1p64f)) || top_p != top_p || min_p != min_p || u != u ||
            most >= KEY_INF || most <= KEY_NONE)
            return false;
        k = greedy ? 1u : top_k > 0 ? (uint32_t)top_k : 0xFFFFFFFFu;
        u = u < 0.0f ? 0.0f : u > 0x1.fffffep-1f ? 0x1.fffffep-1f : u;
        min_p = min_p < 1.0f ? min_p : 1.0f;
        last = min_p > 0.0f ? -32.0 * log2((double)min_p) : __builtin_inf();
        sc.m = sp_value(most);
        sc.c = 32.0 * 1.44269504088896340736 / (greedy ? 1.0 : (double)temperature);
        const int bits = 62 - (32 - __builtin_clz(((uint32_t)vocab - 1u) | 1u));  // (vocab 2^bits stays below 2^63)
        sc.bits = bits < 50 ? bits : 50;
        sc.one = ldexp(1.0, sc.bits);
        return true;
    }
    SYN_DEV Mode mode() const {
        if (k < (uint32_t)vocab && k <= (uint32_t)LIST) return k <= TOP ? LIST_TOP : LIST_K;
        return top_p >= 1.0f && min_p > 0.0f && k >= (uint32_t)vocab ? LIST_MIN_P : BINS;
    }
    // The sum before bin b, of the greatest weight.
    SYN_DEV double base(int b) const { return ldexp((double)r.masses[b], -sc.bits); }

    // (every thread) the greatest of the threads' numbers
    SYN_DEV uint32_t most_of(uint32_t v) {
        if (threadIdx.x == 0) r.most = 0;
        __syncthreads();
        v = group_max_u32<64>(v);
        if ((threadIdx.x & 63) == 0) atomicMax(&r.most, v);
        __syncthreads();
        return r.most;
    }

    // ---- the bins -------------------------------------------------------------------------------------------
    SYN_DEV float s32(float v) const { return ((float)sc.m - v) * (float)sc.c; }
    SYN_DEV int bin32(float v) const {
        const float s = s32(v);
        return s < (float)(SB - 1) ? (int)s : SB - 1;
    }
    // (what is beyond the last bin is counted by each thread: of a cold row it is most, and a bin's sums are added one lane
    // after the other.  A row of 128256 BF16 with a third there 171 us, 60 so)
    SYN_DEV void add_to_bin(float v, uint32_t& beyond) {
        const double s = sc.s(v);
        if (s < (double)(SB - 1)) {
            const Scale::Part p = sc.inside(s);
            atomicAdd(&r.counts[p.bin], 1u);
            atomicAdd((unsigned long long*)&r.masses[p.bin], (unsigned long long)p.whole);
        } else {
            beyond += v > -__builtin_inff() ? 1 : 0;
        }
    }
    // (every thread) each of the weight 2^-64 at most
    SYN_DEV void add_beyond(uint32_t beyond) {
#pragma unroll
        for (int d = 32; d > 0; d /= 2) beyond += __shfl_xor(beyond, d);
        if ((threadIdx.x & 63) == 0 && beyond) {
            const Scale::Part p = sc.part((double)(SB - 1));
            atomicAdd(&r.counts[SB - 1], beyond);
            atomicAdd((unsigned long long*)&r.masses[SB - 1], (unsigned long long)(p.whole * beyond));
        }
        __syncthreads();
    }
    SYN_DEV void no_bins() {
        for (int i = threadIdx.x; i < SB; i += ST) r.counts[i] = 0, r.masses[i] = 0;
        __syncthreads();
    }
    // The counts (and sums) of the bins over this workgroup's values.
    SYN_DEV void bins(Mode mode) {
        no_bins();
        uint32_t beyond = 0;
        if (mode == LIST_K)
            each([&](float v, int) {
                const float s = s32(v);
                if (s < (float)(SB - 1))
                    atomicAdd(&r.counts[(int)s], 1u);
                else
                    beyond += v > -__builtin_inff() ? 1 : 0;
            });
        else
            each([&](float v, int) { add_to_bin(v, beyond); });
        add_beyond(beyond);
    }
    // (every thread) The counts and sums of the bins before each, in place.  (A bin's sum to the nearest whole number: where
    // it is below half of 1 nothing is added, and no sum that is looked for lies there.)
    SYN_DEV void prefix() {
        static_assert(SB == 2 * ST, "two bins a thread");
        const int l = threadIdx.x & 63, wave = threadIdx.x >> 6, b = 2 * (int)threadIdx.x;
        const uint32_t c0 = r.counts[b], c1 = r.counts[b + 1];
        const uint64_t m0 = (uint64_t)__builtin_rint((double)r.masses[b] * Scale::step(b));
        const uint64_t m1 = (uint64_t)__builtin_rint((double)r.masses[b + 1] * Scale::step(b + 1));
        uint32_t n = c0 + c1;
        uint64_t s = m0 + m1;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t on = __shfl_up(n, d);
            const uint64_t os = __shfl_up((unsigned long long)s, d);
            n += l >= d ? on : 0u;
            s += l >= d ? os : 0ull;
        }
        if (l == 63) r.part_n[wave] = n, r.part_s[wave] = s;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < ST / 64; ++w) {
            n += w < wave ? r.part_n[w] : 0u;
            s += w < wave ? r.part_s[w] : 0ull;
        }
        if (threadIdx.x == ST - 1) r.counts[SB] = n, r.masses[SB] = s;
        n -= c0 + c1, s -= m0 + m1;
        r.counts[b] = n, r.masses[b] = s;
        r.counts[b + 1] = n + c0, r.masses[b + 1] = s + m0;
        __syncthreads();
    }
    // (one wavefront) The first bin whose values reach what is wanted (the last that holds any where none does).
    SYN_DEV int bin_of(Want want, uint32_t n, double sum) const {
        const int l = threadIdx.x & 63;
        auto so = [&](int b) { return want == AT_LEAST_N ? r.counts[b + 1] >= n : want == SUM_REACHES ? base(b + 1) >= sum : base(b + 1) > sum; };
        uint64_t yes = __builtin_amdgcn_ballot_w64(so(32 * l + 31));
        if (yes == 0) {
            want = AT_LEAST_N, n = r.counts[SB];
            yes = __builtin_amdgcn_ballot_w64(so(32 * l + 31));
        }
        const int o = 32 * (__builtin_ffsll((long long)yes) - 1);
        return o + __builtin_ffsll((long long)__builtin_amdgcn_ballot_w64(l < 32 && so(o + (l & 31)))) - 1;
    }

    // ---- what to gather -------------------------------------------------------------------------------------
    // Into r.want.  LIST_TOP: from 1024 numbers in r.run's place, each the greatest of a part of the row.
    SYN_DEV void want_top() {
        if (threadIdx.x < 64) {
            const uint32_t* tops = reinterpret_cast<const uint32_t*>(r.run);
            uint32_t of[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                of[j] = 0;
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const uint32_t v = tops[256 * m + 64 * j + threadIdx.x];
                    of[j] = v > of[j] ? v : of[j];
                }
            }
            const uint32_t b = reached_by(of, (int)k);
            Wanted w{};
            w.b = w.cut = -1;
            w.lo = b > KEY_NONE ? sp_value(b) : sp_value(KEY_NONE + 1);
            w.to = b > KEY_NONE ? sc.s(w.lo) : (double)(SB - 1);
            w.hi = w.lo2 = w.hi2 = __builtin_inff();
            if (threadIdx.x == 0) r.want = w;
        }
        __syncthreads();
    }
    // Of the other modes, from the bins (which are prefixes behind it).
    SYN_DEV void want(Mode mode) {
        if (mode != LIST_MIN_P) prefix();
        if (threadIdx.x < 64) {
            Wanted w = wanted(mode);
            edges(mode, w);
            if (threadIdx.x == 0) r.want = w;
        }
        __syncthreads();
    }
    // (one wavefront) The least values of the bins from a1, a0 - 1, b and b - 1 up, the wanted ones' edges, 16 lanes an edge: by
    // 16 numbers at a time between one that is below and one that is not, at first the eight on either side of where the
    // edge lies in 64 bits, where it lies among them (it does but for the rounding of F32 distances).
    SYN_DEV void edges(Mode mode, Wanted& w) const {
        const int l = threadIdx.x & 63, group = l >> 4;
        const int at = group == 0 ? w.a1 : group == 1 ? (mode == BINS ? w.a0 - 1 : -1) : w.b < 0 ? -1 : group == 2 ? w.b : w.b - 1;
        auto in = [&](uint32_t key) {
            const float v = sp_value(key);
            return mode == LIST_MIN_P ? sc.s(v) <= last : (mode == LIST_K ? bin32(v) : Scale::bin(sc.s(v))) <= at;
        };
        const uint32_t top = sp_order((float)sc.m);
        const double s = mode == LIST_MIN_P ? last : (double)at + (mode == LIST_K ? 1.0 : 0.5);
        const uint32_t near = sp_order((float)(sc.m - s / sc.c));
        uint32_t lo = near > KEY_NONE + 8 ? near - 8 : KEY_NONE, hi = near + 8 < top ? near + 8 : top;
        if (lo > KEY_NONE && (lo >= top || in(lo))) lo = KEY_NONE;
        if (hi <= lo || !in(hi)) hi = top;
        if (at < 0 && mode != LIST_MIN_P) lo = hi - 1;  // (none)
#pragma unroll 1
        for (int i = 0; i < 9 && __builtin_amdgcn_ballot_w64(hi - lo > 1) != 0; ++i) {
            const uint32_t step = (hi - lo + 15) >> 4, up = lo + step * (uint32_t)((l & 15) + 1);
            const uint32_t t = up < hi && up > lo ? up : hi;
            const uint32_t yes = (uint32_t)(__builtin_amdgcn_ballot_w64(in(t) || t == hi) >> (16 * group)) & 0xFFFFu;
            const int f = __builtin_ctz(yes);
            const uint32_t to = lo + step * (uint32_t)(f + 1);
            hi = to < hi && to > lo ? to : hi;
            lo = f ? lo + step * (uint32_t)f : lo;
        }
        const float e = at < 0 && mode != LIST_MIN_P ? __builtin_inff() : sp_value(hi);
        w.lo = __shfl(e, 0), w.hi = mode == BINS ? __shfl(e, 16) : __builtin_inff();
        w.lo2 = mode == BINS ? __shfl(e, 32) : __builtin_inff(), w.hi2 = mode == BINS ? __shfl(e, 48) : __builtin_inff();
    }
    SYN_DEV Wanted wanted(Mode mode) const {
        Wanted w{};
        w.b = w.cut = -1;
        w.to = last;
        if (mode == LIST_MIN_P) return w;
        w.n = (uint32_t)LIST + 1;
        if (mode == LIST_K) {
            w.a1 = bin_of(AT_LEAST_N, k, 0.0);
            w.n = r.counts[w.a1 + 1];
            w.to = (double)w.a1 + 1.0;
            return w;
        }
        if (k < r.counts[SB]) return w;  // (a top-k longer than a list: its border, then the others', in seldom())
        const double all = base(SB);
        int p = SB, m = SB;
        if (top_p < 1.0f) p = bin_of(SUM_REACHES, 0, (double)top_p * all);
        if (min_p > 0.0f) m = Scale::bin(last);
        // (of two borders in different bins the first counts)
        if (p < SB || m < SB) {
            w.cut = p < m ? p : m;
            w.by_p = p == w.cut;
            w.by_min_p = m == w.cut;
        }
        // the token's sum lies between these, and its bin so
        const double lo = w.cut >= 0 ? base(w.cut) : all, hi = w.cut >= 0 ? base(w.cut + 1) : all;
        w.a0 = bin_of(SUM_PASSES, 0, (double)u * lo);
        w.a1 = w.cut >= 0 ? bin_of(SUM_PASSES, 0, (double)u * hi) : w.a0;
        if (w.a0 > w.a1) w.a0 = w.a1;
        if (w.cut >= 0) {
            if (w.cut <= w.a1 + 1)
                w.a1 = w.cut > w.a1 ? w.cut : w.a1;
            else
                w.b = w.cut;
        }
        w.n0 = (int)(r.counts[w.a1 + 1] - r.counts[w.a0]);
        w.n = (uint32_t)w.n0 + (w.b >= 0 ? r.in(w.b) : 0);
        w.total = r.counts[SB], w.all = all;
        w.sum0 = base(w.a0);
        w.end = (int)w.n;
        if (w.b >= 0) w.sum1 = base(w.b);
        if (w.cut >= 0) {
            w.i0 = w.b >= 0 ? w.n0 : (int)(r.counts[w.cut] - r.counts[w.a0]);
            w.end = w.i0 + (int)r.in(w.cut);
            w.before = r.counts[w.cut], w.under = base(w.cut);
            if (w.n > (uint32_t)LIST && r.in(w.cut) <= (uint32_t)LIST) {
                w.only = true;
                w.a0 = w.a1 = w.cut, w.b = -1;
                w.i0 = 0, w.end = w.n0 = (int)r.in(w.cut), w.n = r.in(w.cut);
                w.sum0 = w.under;
            }
        }
        return w;
    }
    // The keys of the wanted among this workgroup's values into r.keys, those that find room; r.n: how many there are.
    SYN_DEV void pick(Mode mode) {
        const Wanted& w = r.want;
        if (threadIdx.x == 0) r.n = 0;
        __syncthreads();
        auto put = [&](float v, int i) {
            const uint32_t to = atomicAdd(&r.n, 1u);
            if (to < (uint32_t)LIST) r.keys[to] = sp_key(v, i);
        };
        // (A wavefront whose values are all outside goes on; else each lane puts its own few, mostly one, in turn.)
        auto look = [&](auto&& in) {
            this->pieces(
                [&](u32x4 p, int i) {
                    const uint32_t w0 = p[0], w1 = p[1], w2 = p[2], w3 = p[3];
                    uint32_t mine = 0;
#pragma unroll
                    for (int j = 0; j < Reader<TY>::PER; ++j) mine |= in(this->value(p, j)) ? 1u << j : 0u;
#pragma unroll 1
                    for (; mine != 0; mine &= mine - 1) {
                        const int j = __builtin_ctz(mine), wj = TY == T_F32 ? j : j / 2;
                        const uint32_t a = wj & 1 ? w1 : w0, b = wj & 1 ? w3 : w2;
                        uint32_t one = wj & 2 ? b : a;
                        if constexpr (TY != T_F32) one = j & 1 ? one >> 16 : one;
                        put(TY == T_F32 ? u2f(one) : TY == T_F16 ? f16_to_f32(one) : u2f(one << 16), i + j);
                    }
                },
                [&](float v, int i) {
                    if (in(v)) put(v, i);
                });
        };
        const float lo = w.lo, hi = w.hi, lo2 = w.lo2, hi2 = w.hi2;
        if (mode != BINS)
            look([&](float v) { return v >= lo; });
        else if (w.b < 0)
            look([&](float v) { return v >= lo && v < hi; });
        else
            look([&](float v) { return (v >= lo && v < hi) || (v >= lo2 && v < hi2); });
        __syncthreads();
    }

    // ---- the list -------------------------------------------------------------------------------------------
    // (every thread) r.keys[0 .. n - 1] into order, and their weights into r.run.
    // Up to 64 keys by counting the smaller ones.  More are dealt out to 1024 buckets first, and each counts the smaller
    // ones of its bucket, which are few: buckets of their distances, the wanted bins side by side (from `from` to
    // `to`, the second range moved by `skip`); or, of values of 16 bits (F32 ones may be such), which stand in a bin
    // by the hundred each, buckets of each value's indexes.  (1164 F32 keys 3 us, by compare and exchange 13; 900 of
    // BF16 14 by distances alone.  `to` far from the last one's distance leaves most in one bucket: with one bin for a
    // top-k of 64, some 75 keys, one row of 32064 took 16.2 us in place of 12.7.)
    SYN_DEV void order(int n, double from, double skip, double to) {
        const int i = threadIdx.x;
        if (n <= 64) {
            if (i < 64) {
                const uint64_t mine = i < n ? r.keys[i] : ~0ull;
                r.keys[i] = mine;
                wave_lds_sync();
                int c = 0;
                const ulonglong2* other = reinterpret_cast<const ulonglong2*>(r.keys);
#pragma unroll 8
                for (int j = 0; j < 32; ++j) {
                    const ulonglong2 o = other[j];
                    c += (o.x < mine ? 1 : 0) + (o.y < mine ? 1 : 0);
                }
                wave_lds_sync();
                if (i < n) r.keys[c] = mine, r.run[c] = sc.weight(sc.s(sp_of_key(mine)));
            }
            __syncthreads();
            return;
        }
        const double scale = (double)ST / (to - from);
        constexpr int SHIFT = TY == T_F16 ? 13 : 16;  // of what a value of 16 bits does not have
        uint64_t mine[2];
        uint32_t place[2];
        int bucket[2];
        double at[2];
        bool second[2];
        r.buckets[i] = 0;
        if (i < 5) r.ends[i] = i & 1 ? 0u : 0xFFFFFFFFu;  // the least and greatest of both ranges, whether any is longer
        __syncthreads();
        uint32_t least[2] = {0xFFFFFFFFu, 0xFFFFFFFFu}, most[2] = {0, 0};
        bool longer = false;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (i + ST * m >= n) continue;
            mine[m] = r.keys[i + ST * m];
            const uint32_t key = (uint32_t)(mine[m] >> 32), rest = key & ((1u << SHIFT) - 1u), v = key >> SHIFT;
            longer |= ((rest + 1u) & ((1u << SHIFT) - 1u)) > 1u;  // (all ones above 0, none below)
            const double s = sc.s(sp_of_key(mine[m]));
            second[m] = s > to - 0.5;  // (it begins 1 behind the first's end at least)
            at[m] = ((second[m] ? s - skip : s) - from) * scale;
            second[m] = second[m] && skip > 0.0;
            const int w = second[m] ? 1 : 0;
            least[w] = v < least[w] ? v : least[w], most[w] = v > most[w] ? v : most[w];
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            least[w] = group_min_u32<64>(least[w]), most[w] = group_max_u32<64>(most[w]);
            if ((i & 63) == 0 && least[w] <= most[w]) atomicMin(&r.ends[2 * w], least[w]), atomicMax(&r.ends[2 * w + 1], most[w]);
        }
        if (__builtin_amdgcn_ballot_w64(longer) != 0 && (i & 63) == 0) r.ends[4] = 0;
        __syncthreads();
        const uint32_t l0 = r.ends[0], n_first = l0 <= r.ends[1] ? r.ends[1] - l0 + 1 : 0, l1 = r.ends[2],
                       values = n_first + (l1 <= r.ends[3] ? r.ends[3] - l1 + 1 : 0);
        const uint32_t share = r.ends[4] != 0 && values <= (uint32_t)ST / 2 ? (uint32_t)ST / values : 0;  // a value's buckets
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (i + ST * m >= n) continue;
            if (share) {
                const uint32_t v = (uint32_t)(mine[m] >> 32) >> SHIFT, of = second[m] ? n_first + (v - l1) : v - l0;
                bucket[m] = (int)(of * share + (uint32_t)((uint64_t)(uint32_t)mine[m] * share / (uint32_t)vocab));
            } else {
                bucket[m] = at[m] < (double)(ST - 1) ? (int)(at[m] > 0.0 ? at[m] : 0.0) : ST - 1;
            }
            place[m] = atomicAdd(&r.buckets[bucket[m]], 1u);
        }
        __syncthreads();
        uint32_t up = r.buckets[i];
        const uint32_t own = up;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t o = __shfl_up(up, d);
            up += (i & 63) >= d ? o : 0u;
        }
        if ((i & 63) == 63) r.part_n[i >> 6] = up;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < ST / 64; ++w) up += w < (i >> 6) ? r.part_n[w] : 0u;
        r.buckets[i] = up - own;
        if (i == 0) r.buckets[ST] = (uint32_t)n;
        __syncthreads();
        uint64_t* dealt = reinterpret_cast<uint64_t*>(r.run);
#pragma unroll
        for (int m = 0; m < 2; ++m)
            if (i + ST * m < n) dealt[r.buckets[bucket[m]] + place[m]] = mine[m];
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            if (i + ST * m >= n) continue;
            const uint32_t b0 = r.buckets[bucket[m]], b1 = r.buckets[bucket[m] + 1];
            uint32_t c = b0;
            for (uint32_t j = b0; j < b1; ++j) c += dealt[j] < mine[m] ? 1u : 0u;
            place[m] = c;
        }
        __syncthreads();
#pragma unroll
        for (int m = 0; m < 2; ++m)
            if (i + ST * m < n) r.keys[place[m]] = mine[m], r.run[place[m]] = sc.weight(sc.s(sp_of_key(mine[m])));
        __syncthreads();
    }
    // (one wavefront) The weights' running sums; a lane takes an odd number of neighbours.
    static SYN_DEV int share(int n) { return ((n + 63) / 64) | 1; }
    SYN_DEV void run_up(int n) {
        const int l = threadIdx.x & 63, each = share(n), i0 = l * each, i1 = i0 + each < n ? i0 + each : n;
        double s = 0.0;
        for (int i = i0; i < i1; ++i) s += r.run[i];
        double up = s;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double o = __shfl_up(up, d);
            up += l >= d ? o : 0.0;
        }
        s = __shfl_up(up, 1);
        s = l ? s : 0.0;
        for (int i = i0; i < i1; ++i) {
            s += r.run[i];
            r.run[i] = s;
        }
        wave_lds_sync();
    }
    // (one wavefront) The first of the list's places a .. b - 1 from which on it is so; b where it is of none.
    template <class F>
    SYN_DEV int first(int n, int a, int b, F&& so) const {
        const int l = threadIdx.x & 63, each = share(n);
        const int e = l * each + each < b ? l * each + each - 1 : b - 1;  // the lane's last place
        const uint64_t yes = __builtin_amdgcn_ballot_w64(e >= a && so(e));
        if (yes == 0) return b;
        const int i = (__builtin_ffsll((long long)yes) - 1) * each + l;
        const uint64_t in = __builtin_amdgcn_ballot_w64(l < each && i >= a && i < b && so(i));
        return i - l + __builtin_ffsll((long long)in) - 1;
    }

    // ---- the results ----------------------------------------------------------------------------------------
    SYN_DEV void write(const SampleArgs& g, uint64_t row, uint32_t kept, double w, uint64_t key) const {
        if (threadIdx.x != 0) return;
        g.token[row] = (int)(uint32_t)key;
        g.kept[row] = (int)kept;
        const float lp = (float)(sc.s(sp_of_key(key)) * (-0.69314718055994530942 / 32.0) - log(w));
        g.logprob[row] = kept == 1 || lp > 0.0f ? 0.0f : lp;
    }
    static SYN_DEV void write_none(const SampleArgs& g, uint64_t row) {
        if (threadIdx.x == 0) g.token[row] = -1, g.logprob[row] = __builtin_nanf(""), g.kept[row] = 0;
    }
    // The row's results from the n wanted values, which this workgroup gathers now or which are in r.keys; the sums by one
    // wavefront.  Where they are more than LIST, from the bins and the row.
    SYN_DEV void finish(const SampleArgs& g, uint64_t row, Mode mode, uint32_t n, bool there) {
#pragma unroll 1
        for (;;) {
            if (!there && n <= (uint32_t)LIST) {
                pick(mode);
                n = r.n;
            }
            if (n > (uint32_t)LIST) {
                seldom(g, row, mode);
                return;
            }
            if (mode == BINS) {  // (bin b after a1: nothing between them)
                const int a1 = r.want.a1, b = r.want.b;
                order((int)n, (double)r.want.a0 - 0.5, b >= 0 ? (double)(b - a1 - 1) : 0.0, (double)a1 + (b >= 0 ? 1.5 : 0.5));
            } else {
                order((int)n, 0.0, 0.0, r.want.to);
            }
            const bool only = r.want.only;
            if (only) __syncthreads();
            if (threadIdx.x < 64) results(g, row, mode, n);
            if (!only) return;
            __syncthreads();
            if (!r.at) return;
            n = r.want.n, there = false;
        }
    }
    // (one wavefront) From the list; of `only` the border's bin, the token too if it lies there, else what holds it is wanted
    // next (r.at).
    SYN_DEV void results(const SampleArgs& g, uint64_t row, Mode mode, uint32_t n) {
        run_up((int)n);
        const Wanted& w = r.want;
        const bool bins = mode == BINS, cut = !bins || w.cut >= 0;
        const int n0 = bins ? w.n0 : (int)n, i0 = w.i0;
        int end = bins ? w.end : k < n ? (int)k : (int)n;
        const double sum1 = w.sum1 - (n0 && w.b >= 0 ? r.run[n0 - 1] : 0.0);
        auto run = [&](int i) { return (i < n0 ? w.sum0 : sum1) + r.run[i]; };
        if (cut && top_p < 1.0f && (!bins || w.by_p) && end > i0) {
            const double reach = (double)top_p * (bins ? w.all : run(end - 1));
            const int at = first((int)n, i0, end, [&](int i) { return run(i) >= reach; });
            end = at < end ? at + 1 : end;
        }
        if (cut && min_p > 0.0f && (!bins || w.by_min_p))
            end = first((int)n, i0, end, [&](int i) { return sc.s(sp_of_key(r.keys[i])) > last; });
        const uint32_t kept = cut ? w.before + (uint32_t)(end - i0) : w.total;
        const double all = !cut ? w.all : end > i0 ? run(end - 1) : w.under;
        // (where nothing of the cut's own bin is kept, the token lies in the first range)
        const double pass = (double)u * all;
        if (w.only) {
            const bool next = pass < w.under;
            if (threadIdx.x == 0) r.at = next;
            if (next) {
                Wanted t{};
                t.b = t.cut = -1;
                t.a0 = t.a1 = bin_of(SUM_PASSES, 0, pass);
                t.n = r.in(t.a0), t.n0 = t.end = (int)t.n;
                t.sum0 = base(t.a0);
                t.total = kept, t.all = all;
                edges(mode, t);
                if (threadIdx.x == 0) r.want = t;
                return;
            }
        }
        const int stop = end > 0 ? end : 1, at = first((int)n, 0, stop, [&](int i) { return run(i) > pass; });
        write(g, row, kept, all, r.keys[at < stop ? at : stop - 1]);
    }

    // Where what is wanted is, in its bin: by the list of the bin's values, or where they are too many for one digit by
    // digit of their keys.
    SYN_DEV Place find(Want want, uint32_t n, double sum) {
        if (threadIdx.x < 64) {
            const int o = bin_of(want, n, sum);
            if (threadIdx.x == 0) r.bin = o, r.n = 0;
        }
        __syncthreads();
        const int b = r.bin;
        if (r.in(b) <= (uint32_t)LIST) {
            every([&](float v, int i) {
                if (v != -__builtin_inff() && Scale::bin(sc.s(v)) == b) r.keys[atomicAdd(&r.n, 1u)] = sp_key(v, i);
            });
            __syncthreads();
            const int m = (int)r.n;
            order(m, (double)b - 0.5, 0.0, (double)b + 0.5);
            if (threadIdx.x < 64) {
                run_up(m);
                const double from = base(b);
                const int at = want == AT_LEAST_N ? (int)(n - r.counts[b]) - 1 : first(m, 0, m, [&](int i) {
                    return want == SUM_REACHES ? from + r.run[i] >= sum : from + r.run[i] > sum;
                });
                const int i = at < m ? at : m - 1;
                if (threadIdx.x == 0) r.place = Place{r.counts[b] + (uint32_t)i + 1, from + r.run[i], r.keys[i]};
            }
        } else {
            digits(b, want, n, sum);
        }
        __syncthreads();
        const Place p = r.place;
        __syncthreads();
        return p;
    }
    SYN_DEV void digits(int b, Want want, uint32_t n, double sum) {
        uint32_t* dcount = reinterpret_cast<uint32_t*>(r.run);  // [256]
        uint64_t* dmass = r.keys;
        const double unit = ldexp(Scale::step(b), -sc.bits);
        if (threadIdx.x == 0) r.prefix = 0, r.before = r.counts[b], r.before_mass = 0;
#pragma unroll 1
        for (int shift = 56; shift >= 0; shift -= 8) {
            if (threadIdx.x < 256) dcount[threadIdx.x] = 0, dmass[threadIdx.x] = 0;
            __syncthreads();
            const uint64_t prefix = r.prefix;
            every([&](float v, int i) {
                if (v == -__builtin_inff()) return;
                const Scale::Part p = sc.part(sc.s(v));
                const uint64_t key = sp_key(v, i);
                if (p.bin != b || (shift < 56 && (key >> (shift + 8)) != prefix)) return;
                atomicAdd(&dcount[key >> shift & 255], 1u);
                atomicAdd((unsigned long long*)&dmass[key >> shift & 255], (unsigned long long)p.whole);
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
                    const double c = base(b) + (double)ms * unit;
                    if (want == AT_LEAST_N ? cn >= n : want == SUM_REACHES ? c >= sum : c > sum) break;
                }
                r.prefix = r.prefix << 8 | (uint32_t)d;
                r.before = at_n, r.before_mass = at_ms;
                if (shift == 0) r.place = Place{at_n + 1, base(b) + (double)(at_ms + dmass[d]) * unit, r.prefix};
            }
            __syncthreads();
        }
    }
    // Border by border: the top-k's, the top-p's, min-p's, the token.
    SYN_DEV void seldom(const SampleArgs& g, uint64_t row, Mode mode) {
        if (mode != BINS) {
            no_bins();
            uint32_t beyond = 0;
            every([&](float v, int) { add_to_bin(v, beyond); });
            add_beyond(beyond);
            prefix();
        }
        Place cut{r.counts[SB], base(SB), 0};
#pragma unroll 1
        for (int step = 0; step < 4; ++step) {
            Want want = AT_LEAST_N;
            uint32_t n = 0;
            double sum = 0.0;
            if (step == 0) {
                if (k >= cut.n) continue;
                n = k;
            } else if (step == 1) {
                if (top_p >= 1.0f) continue;
                want = SUM_REACHES, sum = (double)top_p * cut.sum;
            } else if (step == 2) {
                if (!(min_p > 0.0f)) continue;
                if (threadIdx.x == 0) r.n = 0;
                __syncthreads();
                uint32_t mine = 0;
                every([&](float v, int) { mine += v != -__builtin_inff() && sc.s(v) <= last ? 1 : 0; });
                atomicAdd(&r.n, mine);
                __syncthreads();
                n = r.n;
                __syncthreads();
                if (n >= cut.n) continue;
            } else {
                want = SUM_PASSES, sum = (double)u * cut.sum;
            }
            const Place p = find(want, n, sum);
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
    const uint32_t mine = sp.greatest();
    reinterpret_cast<uint32_t*>(r.run)[threadIdx.x] = mine;
    if (!sp.settle(sp.most_of(mine))) {
        sp.write_none(g, row);
        return;
    }
    const Mode mode = sp.mode();
    if (mode == LIST_K || mode == BINS) sp.bins(mode);
    if (mode == LIST_TOP)
        sp.want_top();
    else
        sp.want(mode);
    sp.finish(g, row, mode, r.want.n, false);
}

// ---- few long rows: a row's parts, a launch a step ------------------------------------------------------------
// A row's share of the workspace: the greatest values of the parts' lanes, how many were gathered, the bins, the list.
constexpr int PARTS = 64;
struct Shared {
    uint32_t tops[PARTS][64];
    uint32_t n;
    uint32_t pad[63];
    Wanted want;  // (by the first part, for the end)
    uint32_t counts[SB];
    uint64_t masses[SB];
    uint64_t keys[LIST];
};
static_assert(sizeof(Wanted) % 8 == 0, "the sums on 8 bytes");

template <int TY>
__global__ __launch_bounds__(ST) void k_sample_most(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    const int part = (int)(blockIdx.x % (uint32_t)parts);
    __shared__ uint32_t tops[ST / 64][64];
    Shared& s = ((Shared*)g.ws)[row];
    for (int i = part * ST + (int)threadIdx.x; i < SB; i += parts * ST) s.counts[i] = 0, s.masses[i] = 0;
    if (part == 0 && threadIdx.x == 0) s.n = 0;
    tops[threadIdx.x >> 6][threadIdx.x & 63] = Reader<TY>(g, row, part, parts).greatest();
    __syncthreads();
    if (threadIdx.x >= 64) return;
    uint32_t m = 0;
#pragma unroll
    for (int w = 0; w < ST / 64; ++w) m = tops[w][threadIdx.x] > m ? tops[w][threadIdx.x] : m;
    s.tops[part][threadIdx.x] = m;
}
// (every thread) The lanes' greatest of all parts into 1024 numbers in r.run's place, and the greatest of all.
template <class S>
SYN_DEV uint32_t gather_tops(S& sp, Row& r, const Shared& s, int parts) {
    uint32_t m = 0;
    for (int i = threadIdx.x; i < 64 * parts; i += ST) {
        const uint32_t v = (&s.tops[0][0])[i];
        m = v > m ? v : m;
    }
    reinterpret_cast<uint32_t*>(r.run)[threadIdx.x] = m;
    return sp.most_of(m);
}
template <int TY>
__global__ __launch_bounds__(ST) void k_sample_bins(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    __shared__ Row r;
    Sampler<TY> sp(g, row, r, (int)(blockIdx.x % (uint32_t)parts), parts);
    Shared& s = ((Shared*)g.ws)[row];
    if (!sp.settle(gather_tops(sp, r, s, parts))) return;
    const Mode mode = sp.mode();
    if (mode != LIST_K && mode != BINS) return;
    sp.bins(mode);
    for (int i = threadIdx.x; i < SB; i += ST)  // (whole numbers: in any order)
        if (r.counts[i]) {
            atomicAdd(&s.counts[i], r.counts[i]);
            if (mode == BINS) atomicAdd((unsigned long long*)&s.masses[i], (unsigned long long)r.masses[i]);
        }
}
// What to gather, from the row's bins or tops.
template <class S>
SYN_DEV void want_shared(S& sp, const Shared& s, Row& r, Mode mode) {
    if (mode == LIST_TOP) {
        sp.want_top();
        return;
    }
    if (mode != LIST_MIN_P) {
        for (int i = threadIdx.x; i < SB; i += ST) r.counts[i] = s.counts[i], r.masses[i] = s.masses[i];
        __syncthreads();
    }
    sp.want(mode);
}
template <int TY>
__global__ __launch_bounds__(ST) void k_sample_pick(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x / (uint32_t)parts;
    __shared__ Row r;
    Sampler<TY> sp(g, row, r, (int)(blockIdx.x % (uint32_t)parts), parts);
    Shared& s = ((Shared*)g.ws)[row];
    if (!sp.settle(gather_tops(sp, r, s, parts))) return;
    const Mode mode = sp.mode();
    want_shared(sp, s, r, mode);
    if (blockIdx.x % (uint32_t)parts == 0 && threadIdx.x < sizeof(Wanted) / 4)
        reinterpret_cast<uint32_t*>(&s.want)[threadIdx.x] = reinterpret_cast<const uint32_t*>(&r.want)[threadIdx.x];
    if (r.want.n > (uint32_t)LIST) return;
    sp.pick(mode);
    // (a place for all of this workgroup's at once: one by one, 24 rows' lists took 7 us more)
    const uint32_t n = r.n;
    if (threadIdx.x == 0) r.at = n ? atomicAdd(&s.n, n) : 0;
    __syncthreads();
    const uint32_t at = r.at;
    for (uint32_t i = threadIdx.x; i < n && i < (uint32_t)LIST; i += ST)
        if (at + i < (uint32_t)LIST) s.keys[at + i] = r.keys[i];
}
template <int TY>
__global__ __launch_bounds__(ST) void k_sample_end(SampleArgs g, int parts) {
    const uint64_t row = blockIdx.x;
    __shared__ Row r;
    Sampler<TY> sp(g, row, r);
    Shared& s = ((Shared*)g.ws)[row];
    if (!sp.settle(gather_tops(sp, r, s, parts))) {
        sp.write_none(g, row);
        return;
    }
    const Mode mode = sp.mode();
    if (threadIdx.x < sizeof(Wanted) / 4)
        reinterpret_cast<uint32_t*>(&r.want)[threadIdx.x] = reinterpret_cast<const uint32_t*>(&s.want)[threadIdx.x];
    __syncthreads();
    const uint32_t n = r.want.n <= (uint32_t)LIST ? s.n : r.want.n;
    if (n <= (uint32_t)LIST)
        for (int i = threadIdx.x; i < (int)n; i += ST) r.keys[i] = s.keys[i];
    if (mode == BINS && (n > (uint32_t)LIST || r.want.only)) {
        for (int i = threadIdx.x; i < SB; i += ST) r.counts[i] = s.counts[i], r.masses[i] = s.masses[i];
        __syncthreads();
        sp.prefix();
    }
    __syncthreads();
    sp.finish(g, row, mode, n, true);
}

// How many workgroups share a row: as many as fill the chip twice, of 8192 values at least.
static int sample_parts(int xtype, int rows, int vocab) {
    if (rows > 128 || vocab <= (xtype == T_F32 ? 32768 : 65536)) return 1;
    const int most = vocab / 8192 < PARTS ? vocab / 8192 : PARTS, parts = 512 / rows;
    return parts < most ? parts : most;
}

uint64_t sample_ws_bytes(int xtype, int rows, int vocab) {
    return sample_parts(xtype, rows, vocab) > 1 ? align_up((uint64_t)rows * sizeof(Shared), 256) : 0;
}

template <int TY>
static void sample_as(const SampleArgs& a, hipStream_t stream) {
    const int parts = sample_parts(a.xtype, a.rows, a.vocab);
    if (parts == 1) {
        constexpr int MOST = 1 << 20;  // (a launch's threads are counted in 32 bits)
        for (int t = 0; t < a.rows; t += MOST) {
            SampleArgs g = a;
            g.rows = a.rows - t < MOST ? a.rows - t : MOST;
            g.x = (const uint8_t*)a.x + (uint64_t)t * a.ldx * Reader<TY>::ES;
            g.u = a.u + t;
            if (a.temperature) g.temperature = a.temperature + t;
            if (a.top_k) g.top_k = a.top_k + t;
            if (a.top_p) g.top_p = a.top_p + t;
            if (a.min_p) g.min_p = a.min_p + t;
            g.token = a.token + t, g.logprob = a.logprob + t, g.kept = a.kept + t;
            hipLaunchKernelGGL(k_sample<TY>, dim3(g.rows), dim3(ST), 0, stream, g);
        }
        return;
    }
    const dim3 all((uint32_t)a.rows * (uint32_t)parts);
    // (no row needs bins where every row's top-k is short)
    const bool top = (!a.top_k && a.top_k0 >= 1 && a.top_k0 <= (int)TOP) || (!a.temperature && a.temperature0 == 0.0f);
    hipLaunchKernelGGL(k_sample_most<TY>, all, dim3(ST), 0, stream, a, parts);
    if (!top) hipLaunchKernelGGL(k_sample_bins<TY>, all, dim3(ST), 0, stream, a, parts);
    hipLaunchKernelGGL(k_sample_pick<TY>, all, dim3(ST), 0, stream, a, parts);
    hipLaunchKernelGGL(k_sample_end<TY>, dim3(a.rows), dim3(ST), 0, stream, a, parts);
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
