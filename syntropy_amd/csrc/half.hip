// y = act(x W^T + bias) gate + residual over F16 or BF16 weights.
// The simple form: a wavefront takes a weight row against up to four tokens, 64 values of K a step, in F32.
#include "half.hpp"
#include "kernels.hpp"

namespace syn {

constexpr int DOT_TOKENS = 4;

template <int WTY>
__global__ __launch_bounds__(256) void k_half_dot(HalfArgs g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = (int)blockIdx.x * 4 + wave, t0 = (int)blockIdx.y * DOT_TOKENS;
    if (n >= g.n_out) return;
    const int nt = g.T - t0 < DOT_TOKENS ? g.T - t0 : DOT_TOKENS;
    const uint16_t* w = g.w + (uint64_t)n * g.ldw;
    float acc[DOT_TOKENS] = {};
    for (int k = lane; k < g.k; k += 64) {
        const float wv = half_at(w, WTY, k);
#pragma unroll
        for (int j = 0; j < DOT_TOKENS; ++j)
            if (j < nt) acc[j] = __builtin_fmaf(wv, half_at(g.x + (uint64_t)(t0 + j) * g.ldx, WTY, k), acc[j]);
    }
#pragma unroll
    for (int j = 0; j < DOT_TOKENS; ++j)
        for (int d = 32; d >= 1; d /= 2) acc[j] += __shfl_xor(acc[j], d);
    if (lane < nt) {
        float v = acc[0];
#pragma unroll
        for (int j = 1; j < DOT_TOKENS; ++j) v = lane == j ? acc[j] : v;
        half_emit(g, t0 + lane, n, v);
    }
}

uint64_t half_ws_bytes(int, int, int, bool) { return 0; }

void launch_half_gemv(const HalfArgs& a, bool, uint8_t*, hipStream_t stream) {
    constexpr int MOST = 65535 * DOT_TOKENS;
    for (int t = 0; t < a.T; t += MOST) {  // (what a grid holds)
        HalfArgs g = a;
        auto at = [&](const void* p, int ty, uint64_t ld) {
            return p ? (const uint8_t*)p + (uint64_t)t * ld * (ty == T_F32 ? 4 : 2) : nullptr;
        };
        g.T = a.T - t < MOST ? a.T - t : MOST;
        g.x = a.x + (uint64_t)t * a.ldx;
        g.gate = at(a.gate, a.gtype, a.ldg);
        g.res = at(a.res, a.rtype, a.ldr);
        g.y = (void*)at(a.y, a.ytype, a.ldy);
        const dim3 grid((g.n_out + 3) / 4, (g.T + DOT_TOKENS - 1) / DOT_TOKENS);
        if (a.wtype == T_F16)
            hipLaunchKernelGGL(k_half_dot<T_F16>, grid, dim3(256), 0, stream, g);
        else
            hipLaunchKernelGGL(k_half_dot<T_BF16>, grid, dim3(256), 0, stream, g);
    }
}

}  // namespace syn
