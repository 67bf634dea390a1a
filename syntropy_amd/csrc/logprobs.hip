// Log probabilities of given tokens, entropy and most probable tokens of each row of logits x [rows][vocab]:
//   z = x scale, m = max z, s = sum exp(z - m);  log p_i = (z_i - m) - log s;
//   H = log s - sum exp(z - m) (z - m) / s;  rank = the number of logits above the token's;
//   the `top` first tokens by (logit descending, index ascending).
// A row with nothing visible (all -infinity) has log probabilities of -infinity and the entropy 0; a NaN or
// +infinity in it makes them NaN.  A NaN orders above everything.
#include "common.hpp"
#include "kernels.hpp"

namespace syn {

namespace {

template <int TY>
SYN_DEV float lp_load(const void* x, uint64_t i) {
    if constexpr (TY == T_F32) return ((const float*)x)[i];
    const uint32_t h = ((const uint16_t*)x)[i];
    return TY == T_F16 ? f16_to_f32(h) : u2f(h << 16);
}
// A whole number that orders as the value does: -0 as +0, every NaN above +infinity.
SYN_DEV uint32_t lp_key(float v) {
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t b = f2u(v + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}

}  // namespace

template <int TY>
__global__ __launch_bounds__(256) void k_logprobs(LogprobArgs g) {
    const uint64_t row = blockIdx.x;
    const uint64_t at = row * g.ldx;
    __shared__ float red[3][4];
    __shared__ uint64_t best[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t = g.wide ? ((const int64_t*)g.tokens)[row] : ((const int32_t*)g.tokens)[row];
    const bool known = t >= 0 && t < g.vocab;
    const float xt = known ? lp_load<TY>(g.x, at + t) : 0.0f;
    // the largest scaled logit (a NaN is met in the sum)
    float m = -__builtin_inff();
    for (int i = threadIdx.x; i < g.vocab; i += 256) m = fmaxf(m, lp_load<TY>(g.x, at + i) * g.scale);
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) red[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    __syncthreads();
    const float base = m == -__builtin_inff() ? 0.0f : m;
    float s = 0.0f, e = 0.0f, above = 0.0f;
    for (int i = threadIdx.x; i < g.vocab; i += 256) {
        const float v = lp_load<TY>(g.x, at + i), d = v * g.scale - base, p = expf(d);
        s += p;
        e += p == 0.0f ? 0.0f : p * d;
        above += v > xt ? 1.0f : 0.0f;
    }
    for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d), e += __shfl_xor(e, d), above += __shfl_xor(above, d);
    if (lane == 0) red[0][wave] = s, red[1][wave] = e, red[2][wave] = above;
    __syncthreads();
    s = (red[0][0] + red[0][1]) + (red[0][2] + red[0][3]);
    e = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    above = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
    const bool none = s == 0.0f;
    const float ls = logf(s);
    if (threadIdx.x == 0) {
        g.logprob[row] = t < 0 ? 0.0f : !known ? __builtin_nanf("") : none ? -__builtin_inff() : (xt * g.scale - base) - ls;
        g.rank[row] = known ? (int)above : -1;
        g.entropy[row] = none ? 0.0f : ls - e / s;
    }
    uint64_t last = ~0ull;
    for (int j = 0; j < g.top; ++j) {
        uint64_t b = 0;
        for (int i = threadIdx.x; i < g.vocab; i += 256) {
            const uint64_t k = (uint64_t)lp_key(lp_load<TY>(g.x, at + i)) << 32 | (0x7FFFFFFFu - (uint32_t)i);
            b = k < last && k > b ? k : b;
        }
        for (int d = 32; d; d >>= 1) {
            const uint64_t o = __shfl_xor((unsigned long long)b, d);
            b = o > b ? o : b;
        }
        if (lane == 0) best[wave] = b;
        __syncthreads();
        for (int w = 0; w < 4; ++w) b = best[w] > b ? best[w] : b;
        __syncthreads();
        last = b;
        if (threadIdx.x == 0) {
            const uint32_t i = 0x7FFFFFFFu - (uint32_t)b;
            g.top_ids[row * g.top + j] = (int32_t)i;
            g.top_logprobs[row * g.top + j] =
                none ? -__builtin_inff() : (lp_load<TY>(g.x, at + i) * g.scale - base) - ls;
        }
    }
}

uint64_t logprob_ws_bytes(int, int, int) { return 0; }

void launch_logprobs(const LogprobArgs& a, hipStream_t stream) {
    if (a.xtype == T_F32)
        hipLaunchKernelGGL(k_logprobs<T_F32>, dim3(a.rows), dim3(256), 0, stream, a);
    else if (a.xtype == T_F16)
        hipLaunchKernelGGL(k_logprobs<T_F16>, dim3(a.rows), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(k_logprobs<T_BF16>, dim3(a.rows), dim3(256), 0, stream, a);
}

}  // namespace syn
