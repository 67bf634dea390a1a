// y = x W^T over int8 weights with a scale a channel, the tokens' rows quantized to int8 with a scale a
// token:
//   a_t = max |x_t|, s_t = a_t / 127, q_t = rint(x_t / s_t);  S = sum_k q_tk w_ok, exact in I32;
//   y_to = (S s_t) s_o + b_o, and the gated form silu(y_t,gate) * y_t,up.
// Here: the rows' codes, the fold of a product whose K was split over workgroups, and the choice of the
// product's kernel (int8_few.hip, int8_gemm.hip).  S is a whole number, so every kernel, split and order of
// the sum gives the same bits.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

// ---- a row's scale and codes ------------------------------------------------------------------------
// One workgroup a row: the row's largest magnitude (as bits: non-negative F32 patterns order as their
// values, a NaN's and an infinity's are the largest), then its codes.  A lane holds NC pieces of eight values
// in registers between the two, all of them in flight at once, so the row is read once; longer rows are read
// twice, the second time from L2.  Rows begin at any value's address: global loads take any alignment.
template <int TY, int THREADS, int NC>
__global__ __launch_bounds__(THREADS) void k_i8_quantize(const void* __restrict__ x, uint64_t ldx, int k,
                                                         int8_t* __restrict__ codes, uint64_t ldc, int kp,
                                                         float* __restrict__ scales) {
    const uint64_t row = blockIdx.x;
    const uint8_t* xr = (const uint8_t*)x + row * ldx * (TY == T_F32 ? 4 : 2);
    int8_t* cr = codes + row * ldc;
    __shared__ uint32_t top[THREADS / 64];
    float v[NC][8];
    uint32_t m = 0;
    if (k <= NC * THREADS * 8) {
#pragma unroll
        for (int c = 0; c < NC; ++c) i8_load8<TY>(xr, (c * THREADS + (int)threadIdx.x) * 8, k, v[c]);
#pragma unroll
        for (int c = 0; c < NC; ++c) m = i8_max8(v[c], m);
    } else {
        for (int i = threadIdx.x * 8; i < k; i += THREADS * 8) {
            i8_load8<TY>(xr, i, k, v[0]);
            m = i8_max8(v[0], m);
        }
    }
    m = group_max_u32<64>(m);
    if ((threadIdx.x & 63) == 0) top[threadIdx.x >> 6] = m;
    __syncthreads();
    for (int w = 0; w < THREADS / 64; ++w) m = m > top[w] ? m : top[w];
    const I8Scale s = i8_scale(m);
    if (threadIdx.x == 0) scales[row] = s.s;
    if (k <= NC * THREADS * 8) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int i = (c * THREADS + (int)threadIdx.x) * 8;
            if (i < kp) *reinterpret_cast<uint2*>(cr + i) = i8_codes8(v[c], s.inv);
        }
    } else {
        for (int i = threadIdx.x * 8; i < kp; i += THREADS * 8) {
            i8_load8<TY>(xr, i, k, v[0]);
            *reinterpret_cast<uint2*>(cr + i) = i8_codes8(v[0], s.inv);
        }
    }
}

template <int TY>
static void quantize_as(const void* x, uint64_t ldx, int rows, int k, int8_t* codes, uint64_t ldc, int kp, float* scales,
                        hipStream_t stream) {
#define SYN_Q(THREADS, NC)                                                                                            \
    hipLaunchKernelGGL((k_i8_quantize<TY, THREADS, NC>), dim3(rows), dim3(THREADS), 0, stream, x, ldx, k, codes, ldc, kp, \
                       scales)
    // few long rows on more threads each: 32 rows of 14336 5.7 us on 1024, 7.7 on 256
    if (kp > 4096 && rows <= 256)
        SYN_Q(1024, 2);
    else if (kp <= 2048)
        SYN_Q(256, 1);
    else if (kp <= 4096)
        SYN_Q(256, 2);
    else if (kp <= 8192)
        SYN_Q(256, 4);
    else
        SYN_Q(256, 8);
#undef SYN_Q
}

void launch_i8_quantize(int xtype, const void* x, uint64_t ldx, int rows, int k, int8_t* codes, uint64_t ldc,
                        float* scales, hipStream_t stream) {
    const int kp = (int)(i8_padded(k) < ldc ? i8_padded(k) : ldc);
    if (xtype == T_F32)
        quantize_as<T_F32>(x, ldx, rows, k, codes, ldc, kp, scales, stream);
    else if (xtype == T_F16)
        quantize_as<T_F16>(x, ldx, rows, k, codes, ldc, kp, scales, stream);
    else
        quantize_as<T_BF16>(x, ldx, rows, k, codes, ldc, kp, scales, stream);
}

// ---- the fold of a split K ----------------------------------------------------------------------------
// An output a lane: its parts added, then the epilogue.
__global__ __launch_bounds__(256) void k_i8_fold(I8Args g) {
    const int n = blockIdx.x * 256 + threadIdx.x, t = blockIdx.y;
    if (n >= g.n_out) return;
    const uint64_t rows_w = (uint64_t)g.n_out * (g.gated ? 2 : 1), part = (uint64_t)g.T * rows_w;
    const int* p = g.partial + (uint64_t)t * rows_w + n;
    int s0 = 0, s1 = 0;
    for (int z = 0; z < g.splits; ++z) {
        s0 += p[z * part];
        if (g.gated) s1 += p[z * part + g.n_out];
    }
    const float sx = g.xs[t];
    float v = i8_value(s0, sx, g.ws[n]);
    if (g.bias) v = v + g.bias[n];
    if (g.gated) {
        float u = i8_value(s1, sx, g.ws[g.n_out + n]);
        if (g.bias) u = u + g.bias[g.n_out + n];
        v = i8_silu(v) * u;
    }
    i8_store(g.y, g.ytype, (uint64_t)t * g.ldy + n, v);
}

static void launch_i8_fold(const I8Args& a, hipStream_t stream) {
    hipLaunchKernelGGL(k_i8_fold, dim3((a.n_out + 255) / 256, a.T), dim3(256), 0, stream, a);
}

// ---- the choice ----------------------------------------------------------------------------------------
bool i8_fused(int rows_w, int k, int T) { return i8_few_fused(rows_w, k, T); }

int i8_splits(int rows_w, int k, int T) { return i8_few_fits(rows_w, T) ? 1 : i8_gemm_pick(rows_w, k, T).splits; }

void launch_i8_gemv(const I8Args& a, hipStream_t stream) {
    const int rows_w = a.n_out * (a.gated ? 2 : 1);
    const I8Pick p = i8_gemm_pick(rows_w, a.k, a.T);
    // (weight rows may be so far apart that a tile's offsets pass 32 bits)
    if (i8_few_fits(rows_w, a.T) || !i8_gemm_reaches(p.tile, a)) {
        launch_i8_few(a, stream);
        return;
    }
    launch_i8_gemm(p.tile, a, stream);
    if (a.splits > 1) launch_i8_fold(a, stream);
}

}  // namespace syn
