// The end of a block and the beginning of the next (no counterpart in the reference, whose RmsNorm is norm.hip):
//   a = post ? rms(branch; post) : branch;  h = x + (scale gate) a;  y = rms(h; g)
//   rms(v; g) = v g / sqrt(mean v^2 + eps)
// in F32: h is rounded to the stream's type once where it is stored, and y comes from the h that is not.
//
// Bound by HBM: x, the branch and a gate of a value an output are read once, h and y written once.  A row lies in
// the registers of the wavefronts that share it, pieces of eight values a lane, so that nothing is read twice
// and h may be x itself.
#include <type_traits>

#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

template <int TY>
SYN_DEV void bn_store8(void* p, uint64_t at, int i, int n, const float (&v)[8]) {
    uint8_t* to = (uint8_t*)p + (at + i) * (TY == T_F32 ? 4 : 2);
    if constexpr (TY == T_F32) {
        if (i + 8 <= n) {
            __builtin_memcpy(to, v, 32);
            return;
        }
    } else {
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = i8_half2<TY>(v[2 * j], v[2 * j + 1]);
        if (i + 8 <= n) {
            __builtin_memcpy(to, h, 16);
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (i + j < n) i8_store(p, TY, at + i + j, v[j]);
}
// The sum over the threads of a row (WAVES wavefronts), the same in each: lanes by halves, then wavefronts in order.
template <int WAVES>
SYN_DEV float bn_sum(float v, float* part) {
    for (int d = 32; d >= 1; d /= 2) v += __shfl_xor(v, d);
    if constexpr (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) s += part[w];
    return s;
}

// P pieces a lane.
template <int TX, int TB, int WAVES, int P>
__global__ __launch_bounds__(64 * WAVES) void k_block_norm(BlockNormArgs g) {
    const uint64_t row = blockIdx.x;
    const int n = g.n;
    __shared__ float part[2][WAVES];
    float h[P][8], a[P][8];
    auto at = [&](int p) { return 8 * ((int)threadIdx.x + 64 * WAVES * p); };
    const uint8_t* x = (const uint8_t*)g.x + row * g.ldx * (TX == T_F32 ? 4 : 2);
#pragma unroll
    for (int p = 0; p < P; ++p) i8_load8<TX>(x, at(p), n, h[p]);
    if (g.branch) {
        const uint8_t* b = (const uint8_t*)g.branch + row * g.ldb * (TB == T_F32 ? 4 : 2);
#pragma unroll
        for (int p = 0; p < P; ++p) i8_load8<TB>(b, at(p), n, a[p]);
        float r = 1.0f;
        if (g.post) {
            float s = 0.0f;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < 8; ++j) s = __builtin_fmaf(a[p][j], a[p][j], s);
            r = 1.0f / sqrtf(bn_sum<WAVES>(s, part[0]) / (float)n + g.eps);
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float w[8];
            if (g.post) {
                i8_load8<T_F32>((const uint8_t*)g.post, at(p), n, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) a[p][j] = a[p][j] * r * w[j];
            }
            if (g.gate) {
                i8_load8<TB>((const uint8_t*)g.gate + row * g.ldg * (TB == T_F32 ? 4 : 2), at(p), n, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) a[p][j] = a[p][j] * w[j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) h[p][j] = __builtin_fmaf(g.scale, a[p][j], h[p][j]);
            if (at(p) < n) bn_store8<TX>(g.h, row * g.ldh, at(p), n, h[p]);
        }
    }
    if (!g.g) return;
    float s = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (at(p) + j < n) s = __builtin_fmaf(h[p][j], h[p][j], s);
    const float r = 1.0f / sqrtf(bn_sum<WAVES>(s, part[1]) / (float)n + g.eps);
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (at(p) >= n) continue;
        float w[8];
        i8_load8<T_F32>((const uint8_t*)g.g, at(p), n, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[p][j] = h[p][j] * r * w[j];
        if (g.ytype == T_F32)
            bn_store8<T_F32>(g.y, row * g.ldy, at(p), n, h[p]);
        else if (g.ytype == T_F16)
            bn_store8<T_F16>(g.y, row * g.ldy, at(p), n, h[p]);
        else
            bn_store8<T_BF16>(g.y, row * g.ldy, at(p), n, h[p]);
    }
}

template <int TX, int TB>
static void launch_typed(const BlockNormArgs& a, hipStream_t stream) {
    if (a.n <= 8 * 64 * 4 * 2)
        hipLaunchKernelGGL((k_block_norm<TX, TB, 4, 2>), dim3(a.rows), dim3(256), 0, stream, a);
    else if (a.n <= 8 * 64 * 16 * 2)
        hipLaunchKernelGGL((k_block_norm<TX, TB, 16, 2>), dim3(a.rows), dim3(1024), 0, stream, a);
    else
        hipLaunchKernelGGL((k_block_norm<TX, TB, 16, 4>), dim3(a.rows), dim3(1024), 0, stream, a);
}
static_assert(8 * 64 * 16 * 4 == BLOCK_NORM_MAX_COLS, "the longest row");

template <int TX>
static void launch_from(const BlockNormArgs& a, hipStream_t stream) {
    if (a.btype == T_F32)
        launch_typed<TX, T_F32>(a, stream);
    else if (a.btype == T_F16)
        launch_typed<TX, T_F16>(a, stream);
    else
        launch_typed<TX, T_BF16>(a, stream);
}

void launch_block_norm(const BlockNormArgs& a, hipStream_t stream) {
    if (a.xtype == T_F32)
        launch_from<T_F32>(a, stream);
    else if (a.xtype == T_F16)
        launch_from<T_F16>(a, stream);
    else
        launch_from<T_BF16>(a, stream);
}

}  // namespace syn
