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
    // what a whole number of bin b stands for
    SYN_DEV double unit(int b) const { return exp2((double)b * (-1.0 / 32.0)) / one; }
};

enum Want { AT_LEAST_N, SUM_REACHES, SUM_PASSES };

struct Row {
    uint32_t count[SB];
    uint64_t mass[SB];
    uint32_t count0[SB + 1];  // before a bin
    double base[SB + 1];
    uint32_t dcount[256];
    uint64_t dmass[256];
    uint32_t most;
    // of descend()
    uint64_t prefix, before_mass;
    uint32_t before;
    uint32_t n;        // the element's place in the order, from 1
    double sum;        // the sum up to it
    uint32_t few;
};

template <int TY>
struct Sampler {
    const uint8_t* x;
    int vocab;
    Scale sc;
    Row& r;

    // The first element of the order whose place or running sum is what is wanted (the last where none is):
    // its bin from the bins' sums, then digit by digit of (order from above, index).
    SYN_DEV void find(Want want, uint32_t n, double sum) {
        int b = SB;
        for (int i = threadIdx.x; i < SB; i += ST) {
            const bool yes = r.count[i] && (want == AT_LEAST_N ? r.count0[i + 1] >= n
                                            : want == SUM_REACHES ? r.base[i + 1] >= sum : r.base[i + 1] > sum);
            if (yes && i < b) b = i;
        }
        if (threadIdx.x == 0) r.few = SB, r.n = 0;
        __syncthreads();
        if (b < SB) atomicMin(&r.few, (uint32_t)b);
        for (int i = threadIdx.x; i < SB; i += ST)
            if (r.count[i]) atomicMax(&r.n, (uint32_t)i);  // (the last bin that holds anything)
        __syncthreads();
        b = r.few < SB ? (int)r.few : (int)r.n;
        const double unit = sc.unit(b);
        __syncthreads();
        if (threadIdx.x == 0) r.prefix = 0, r.before = r.count0[b], r.before_mass = 0;
#pragma unroll 1
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (int i = threadIdx.x; i < 256; i += ST) r.dcount[i] = 0, r.dmass[i] = 0;
            __syncthreads();
            const uint64_t prefix = r.prefix;
            for (int i = threadIdx.x; i < vocab; i += ST) {
                const float v = sp_load<TY>(x, i);
                if (v == -__builtin_inff()) continue;
                const double s = sc.s(v);
                const uint64_t key = (uint64_t)~sp_order(v) << 32 | (uint32_t)i;
                if (Scale::bin(s) != b || (shift < 56 && (key >> (shift + 8)) != prefix)) continue;
                atomicAdd(&r.dcount[key >> shift & 255], 1u);
                atomicAdd((unsigned long long*)&r.dmass[key >> shift & 255], (unsigned long long)sc.whole(s, b));
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                int d = -1;
                uint32_t cn = r.before, at_n = cn;
                uint64_t ms = r.before_mass, at_ms = ms;
                for (int i = 0; i < 256; ++i) {
                    if (!r.dcount[i]) continue;
                    d = i, at_n = cn, at_ms = ms;
                    cn += r.dcount[i], ms += r.dmass[i];
                    const double c = r.base[b] + (double)ms * unit;
                    if (want == AT_LEAST_N ? cn >= n : want == SUM_REACHES ? c >= sum : c > sum) break;
                }
                r.prefix = r.prefix << 8 | (uint32_t)d;
                r.before = at_n, r.before_mass = at_ms;
                if (shift == 0) r.n = at_n + 1, r.sum = r.base[b] + (double)(at_ms + r.dmass[d]) * unit;
            }
            __syncthreads();
        }
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
    for (int i = threadIdx.x; i < SB; i += ST) r.count[i] = 0, r.mass[i] = 0;
    __syncthreads();
    uint32_t most = 0;
    for (int i = threadIdx.x; i < g.vocab; i += ST) {
        const uint32_t k = sp_order(sp_load<TY>(sp.x, i));
        most = k > most ? k : most;
    }
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
    for (int i = threadIdx.x; i < g.vocab; i += ST) {
        const float v = sp_load<TY>(sp.x, i);
        if (v == -__builtin_inff()) continue;
        const double s = sc.s(v);
        const int b = Scale::bin(s);
        atomicAdd(&r.count[b], 1u);
        atomicAdd((unsigned long long*)&r.mass[b], (unsigned long long)sc.whole(s, b));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        uint32_t n = 0;
        double z = 0.0;
        for (int b = 0; b < SB; ++b) {
            r.count0[b] = n, r.base[b] = z;
            n += r.count[b];
            if (r.mass[b]) z += (double)r.mass[b] * sc.unit(b);
        }
        r.count0[SB] = n, r.base[SB] = z;
    }
    __syncthreads();
    uint32_t n = r.count0[SB];
    double w = r.base[SB];
    const uint32_t k = greedy ? 1u : top_k > 0 ? (uint32_t)top_k : n;
    auto cut = [&](Want want, uint32_t an, double as) {
        sp.find(want, an, as);
        n = r.n, w = r.sum;
        __syncthreads();
    };
    if (k < n) cut(AT_LEAST_N, k, 0.0);
    if (top_p < 1.0f) {
        const uint32_t most_n = n;
        const double all = w;
        cut(SUM_REACHES, 0, (double)top_p * all);
        if (n > most_n) n = most_n, w = all;
    }
    if (min_p > 0.0f) {
        min_p = min_p < 1.0f ? min_p : 1.0f;
        const double last = -32.0 * log2((double)min_p);
        if (threadIdx.x == 0) r.few = 0;
        __syncthreads();
        uint32_t mine = 0;
        for (int i = threadIdx.x; i < g.vocab; i += ST) {
            const float v = sp_load<TY>(sp.x, i);
            mine += v != -__builtin_inff() && sc.s(v) <= last ? 1 : 0;
        }
        atomicAdd(&r.few, mine);
        __syncthreads();
        const uint32_t reach = r.few;
        __syncthreads();
        if (reach < n) cut(AT_LEAST_N, reach, 0.0);
    }
    u = u < 0.0f ? 0.0f : u > 0x1.fffffep-1f ? 0x1.fffffep-1f : u;
    sp.find(SUM_PASSES, 0, (double)u * w);
    if (threadIdx.x == 0) {
        const int id = (int)(uint32_t)r.prefix;
        g.token[row] = id;
        g.kept[row] = (int)n;
        const double s = sc.s(sp_load<TY>(sp.x, id));
        const float lp = (float)(-(s * (0.69314718055994530942 / 32.0)) - log(w));
        g.logprob[row] = n == 1 || lp > 0.0f ? 0.0f : lp;
    }
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
