// y = act(x W^T + bias) gate + residual over F16 or BF16 weights: the copy of x's rows to whole lines, the fold of a
// split K, and the choice of the kernels.
#include "half.hpp"
#include "kernels.hpp"

namespace syn {

// ---- rows of x that are no whole lines, once, zeros behind them ---------------------------------------------
// Eight values a thread.
__global__ __launch_bounds__(256) void k_half_rows(const uint16_t* x, uint64_t ldx, int rows, int k, int kp, uint16_t* out) {
    const int pieces = kp / 8;
    const uint64_t id = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint64_t t = id / (uint32_t)pieces;
    const int i = 8 * (int)(id % (uint32_t)pieces);
    if (t >= (uint64_t)rows) return;
    const uint16_t* from = x + t * ldx + i;
    uint32_t h[4] = {};
    if (i + 8 <= k) {
        __builtin_memcpy(h, from, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (i + e < k) h[e / 2] |= (uint32_t)from[e] << (16 * (e & 1));
    }
    *reinterpret_cast<uint4*>(out + t * (uint32_t)kp + i) = uint4{h[0], h[1], h[2], h[3]};
}

// ---- the fold of a split K ----------------------------------------------------------------------------
// Four outputs a thread: their parts added in order, then the epilogue.
__global__ __launch_bounds__(256) void k_half_fold(HalfArgs g) {
    const int n = 4 * ((int)blockIdx.x * 256 + (int)threadIdx.x), t = blockIdx.y;
    if (n >= g.n_out) return;
    const int in = g.n_out - n < 4 ? g.n_out - n : 4;
    const uint64_t part = (uint64_t)g.T * g.n_out;
    const float* p = g.partial + (uint64_t)t * g.n_out + n;
    const HalfRest rest = half_rest(g, t, n, in);
    float sum[4] = {};
    for (int z = 0; z < g.splits; ++z) {
        float v[4];
        half_load<4>(p + z * part, T_F32, 0, in, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += v[e];
    }
    half_emit(g, t, n, in, sum, rest);
}

// ---- the choice ----------------------------------------------------------------------------------------
// A workspace: the rows of x, then the parts' sums.
static uint64_t rows_bytes(int k, int T, bool lines) { return lines ? 0 : align_up(2 * half_padded(k) * (uint64_t)T, 256); }

uint64_t half_ws_bytes(int n_out, int k, int T, bool lines) {
    if (half_few_fits(T)) return 0;
    const uint64_t splits = (uint64_t)half_gemm_pick(n_out, k, T).splits;
    return rows_bytes(k, T, lines) + (splits > 1 ? align_up(4 * splits * (uint64_t)T * (uint64_t)n_out, 256) : 0);
}

void launch_half_gemv(const HalfArgs& in, bool lines, uint8_t* ws, hipStream_t stream) {
    HalfArgs a = in;
    if (half_few_fits(a.T)) {
        launch_half_few(a, stream);
        return;
    }
    const HalfPick p = half_gemm_pick(a.n_out, a.k, a.T);
    if (!lines) {
        const int kp = (int)half_padded(a.k), most = (1 << 30) / (kp / 8);  // (a launch's threads are counted in 32 bits)
        for (int t = 0; t < a.T; t += most) {
            const int rows = a.T - t < most ? a.T - t : most;
            const uint64_t pieces = (uint64_t)rows * (uint64_t)(kp / 8);
            hipLaunchKernelGGL(k_half_rows, dim3((uint32_t)((pieces + 255) / 256)), dim3(256), 0, stream, a.x + (uint64_t)t * a.ldx,
                               a.ldx, rows, a.k, kp, (uint16_t*)ws + (uint64_t)t * (uint64_t)kp);
        }
        a.x = (const uint16_t*)ws;
        a.ldx = (uint64_t)kp;
    }
    // (rows may be so far apart that a tile's offsets pass 32 bits: their sums have the few-token form's order)
    if (!half_gemm_reaches(p.tile, a)) {
        launch_half_few(a, stream);
        return;
    }
    a.splits = p.splits;
    a.partial = p.splits > 1 ? (float*)(ws + rows_bytes(a.k, a.T, lines)) : nullptr;
    launch_half_gemm(p.tile, a, stream);
    if (p.splits > 1)  // (never more rows than a grid holds: K is split where the tiles are few)
        hipLaunchKernelGGL(k_half_fold, dim3((a.n_out + 1023) / 1024, a.T), dim3(256), 0, stream, a);
}

}  // namespace syn
