// y = x W^T over int8 weights with a scale a channel, the tokens' rows quantized to int8 with a scale a
// token:
//   a_t = max |x_t|, s_t = a_t / 127, q_t = rint(x_t / s_t);  S = sum_k q_tk w_ok, exact in I32;
//   y_to = (S s_t) s_o + b_o, and the gated form silu(y_t,gate) * y_t,up.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

// ---- a row's scale and codes ------------------------------------------------------------------------
// One workgroup a row: the row's largest magnitude (as bits: non-negative F32 patterns order as their
// values, a NaN's and an infinity's are the largest), then its codes; the second reading comes from L2.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_i8_quantize(const void* __restrict__ x, int xtype, uint64_t ldx, int k,
                                                         int8_t* __restrict__ codes, uint64_t ldc, int kp,
                                                         float* __restrict__ scales) {
    const uint64_t row = blockIdx.x;
    __shared__ uint32_t top[THREADS / 64];
    uint32_t m = 0;
    for (int i = threadIdx.x; i < k; i += THREADS) {
        const uint32_t b = f2u(i8_load(x, xtype, row * ldx + i)) & 0x7FFFFFFFu;
        m = m > b ? m : b;
    }
    m = group_max_u32<64>(m);
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int w = 0; w < THREADS / 64; ++w) m = m > top[w] ? m : top[w];
    const I8Scale s = i8_scale(m);
    int8_t* cr = codes + row * ldc;
    for (int i = threadIdx.x; i < kp; i += THREADS)
        cr[i] = i < k ? (int8_t)i8_code(i8_load(x, xtype, row * ldx + i), s.inv) : 0;
    if (threadIdx.x == 0) scales[row] = s.s;
}

void launch_i8_quantize(int xtype, const void* x, uint64_t ldx, int rows, int k, int8_t* codes, uint64_t ldc,
                        float* scales, hipStream_t stream) {
    const int kp = (int)(i8_padded(k) < ldc ? i8_padded(k) : ldc);
    hipLaunchKernelGGL(k_i8_quantize<256>, dim3(rows), dim3(256), 0, stream, x, xtype, ldx, k, codes, ldc, kp, scales);
}

// ---- the product, one output a wavefront ------------------------------------------------------------
__global__ __launch_bounds__(256) void k_i8_dot(I8Args g) {
    const int lane = threadIdx.x & 63;
    const int64_t o = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (o >= g.n_out) return;
    const uint64_t kp = i8_padded(g.k);
    for (int t = blockIdx.y; t < g.T; t += gridDim.y) {
        float v[2] = {0.0f, 0.0f};
        for (int m = 0; m <= g.gated; ++m) {
            const int64_t r = o + (int64_t)m * g.n_out;
            const int8_t* wr = g.w + r * g.ldw;
            const int8_t* xr = g.xq + t * kp;
            int s = 0;
            for (int i = lane; i < g.k; i += 64) s += (int)wr[i] * (int)xr[i];
            for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
            v[m] = i8_value(s, g.xs[t], g.ws[r]);
            if (g.bias) v[m] = v[m] + g.bias[r];
        }
        if (lane == 0) i8_store(g.y, g.ytype, (uint64_t)t * g.ldy + o, g.gated ? ref_silu(v[0]) * v[1] : v[0]);
    }
}

bool i8_fused(int, int, int, int) { return false; }
int i8_splits(int, int, int, int) { return 1; }

void launch_i8_gemv(const I8Args& a, hipStream_t stream) {
    const int ny = a.T < 65535 ? a.T : 65535;
    hipLaunchKernelGGL(k_i8_dot, dim3((a.n_out + 3) / 4, ny), dim3(256), 0, stream, a);
}

}  // namespace syn
