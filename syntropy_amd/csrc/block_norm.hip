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

constexpr int BN_ROWS = 4;

// P pieces a lane.  What is multiplied behind a sum over the row is loaded before it: behind it each load would wait
// for memory with nothing beside it (333 rows of 2011 with all of them 6.9 us so, 6.4 this way).
template <int TX, int TB, int WAVES, int P>
__global__ __launch_bounds__(64 * (WAVES > 1 ? WAVES : BN_ROWS)) void k_block_norm(BlockNormArgs g) {
    // (a wavefront a row: some rows a workgroup, which need nothing of one another)
    const uint64_t row = WAVES > 1 ? blockIdx.x : (uint64_t)blockIdx.x * BN_ROWS + (threadIdx.x >> 6);
    if (WAVES == 1 && row >= (uint64_t)g.rows) return;
    const int n = g.n, lane = WAVES > 1 ? (int)threadIdx.x : (int)(threadIdx.x & 63);
    __shared__ float part[2][WAVES];
    float h[P][8], w[P][8];
    auto at = [&](int p) { return 8 * (lane + 64 * WAVES * p); };
    auto weights = [&](const float* v) {
#pragma unroll
        for (int p = 0; p < P; ++p) i8_load8<T_F32>((const uint8_t*)v, at(p), n, w[p]);
    };
    const uint8_t* x = (const uint8_t*)g.x + row * g.ldx * (TX == T_F32 ? 4 : 2);
    if (g.branch) {
        float a[P][8];
        const uint8_t* b = (const uint8_t*)g.branch + row * g.ldb * (TB == T_F32 ? 4 : 2);
        const uint8_t* gate = g.gate ? (const uint8_t*)g.gate + row * g.ldg * (TB == T_F32 ? 4 : 2) : b;
        float gv[P][8];
#pragma unroll
        for (int p = 0; p < P; ++p) i8_load8<TB>(b, at(p), n, a[p]);
        if (g.post) weights(g.post);
#pragma unroll
        for (int p = 0; p < P; ++p) i8_load8<TB>(gate, at(p), n, gv[p]);
#pragma unroll
        for (int p = 0; p < P; ++p) i8_load8<TX>(x, at(p), n, h[p]);
        if (g.post) {
            float s = 0.0f;
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < 8; ++j) s = __builtin_fmaf(a[p][j], a[p][j], s);
            const float r = 1.0f / sqrtf(bn_sum<WAVES>(s, part[0]) / (float)n + g.eps);
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
                for (int j = 0; j < 8; ++j) a[p][j] = a[p][j] * r * w[p][j];
        }
        if (g.g) weights(g.g);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            if (g.gate) {
#pragma unroll
                for (int j = 0; j < 8; ++j) a[p][j] = a[p][j] * gv[p][j];
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) h[p][j] = __builtin_fmaf(g.scale, a[p][j], h[p][j]);
            if (at(p) < n) bn_store8<TX>(g.h, row * g.ldh, at(p), n, h[p]);
        }
    } else {
#pragma unroll
        for (int p = 0; p < P; ++p) i8_load8<TX>(x, at(p), n, h[p]);
        weights(g.g);
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
#pragma unroll
        for (int j = 0; j < 8; ++j) h[p][j] = h[p][j] * r * w[p][j];
        if (g.ytype == T_F32)
            bn_store8<T_F32>(g.y, row * g.ldy, at(p), n, h[p]);
        else if (g.ytype == T_F16)
            bn_store8<T_F16>(g.y, row * g.ldy, at(p), n, h[p]);
        else
            bn_store8<T_BF16>(g.y, row * g.ldy, at(p), n, h[p]);
    }
}

template <int TX, int TB, int WAVES, int P>
static void launch_as(const BlockNormArgs& a, hipStream_t stream) {
    constexpr int ROWS = WAVES > 1 ? 1 : BN_ROWS, MOST = 1 << 20;  // (a launch's threads are counted in 32 bits)
    auto at = [](const void* p, int ty, uint64_t ld, int t) {
        return p ? (const uint8_t*)p + (uint64_t)t * ld * (ty == T_F32 ? 4 : 2) : nullptr;
    };
    for (int t = 0; t < a.rows; t += MOST) {
        BlockNormArgs g = a;
        g.rows = a.rows - t < MOST ? a.rows - t : MOST;
        g.x = at(a.x, TX, a.ldx, t);
        g.branch = at(a.branch, TB, a.ldb, t);
        g.gate = at(a.gate, TB, a.ldg, t);  // (ldg 0: one for all)
        g.h = (void*)at(a.h, TX, a.ldh, t);
        g.y = (void*)at(a.y, a.ytype, a.ldy, t);
        hipLaunchKernelGGL((k_block_norm<TX, TB, WAVES, P>), dim3((g.rows + ROWS - 1) / ROWS), dim3(64 * WAVES * ROWS), 0, stream, g);
    }
}
// As many wavefronts as hold a row in one or two pieces a lane: more rows are in flight than with more pieces or with more
// wavefronts (2048 rows of 8192 on 16 wavefronts 44 us, on 8 31; 32768 of 512 on four 89, on one 26).
template <int TX, int TB>
static void launch_typed(const BlockNormArgs& a, hipStream_t stream) {
    constexpr int PIECE = 8 * 64;
    if (a.n <= PIECE)
        launch_as<TX, TB, 1, 1>(a, stream);
    else if (a.n <= 2 * PIECE)
        launch_as<TX, TB, 1, 2>(a, stream);
    else if (a.n <= 4 * PIECE)
        launch_as<TX, TB, 4, 1>(a, stream);
    else if (a.n <= 8 * PIECE)
        launch_as<TX, TB, 4, 2>(a, stream);
    else if (a.n <= 16 * PIECE)
        launch_as<TX, TB, 8, 2>(a, stream);
    else if (a.n <= 32 * PIECE)
        launch_as<TX, TB, 16, 2>(a, stream);
    else
        launch_as<TX, TB, 16, 4>(a, stream);
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
