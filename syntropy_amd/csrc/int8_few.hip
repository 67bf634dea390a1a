// The int8 product at few tokens (one to 32): bound by reading the weights once from HBM.
//
// v_mfma_i32_16x16x64_i8 takes 16 weight rows against 16 tokens, 64 values a step.  A lane loads its operand's
// 16 codes straight from the weight row to registers (four lanes a row: 64 bytes of each of 16 rows an
// instruction), since no other wavefront reads them.  The wavefronts of a workgroup share 16 RT rows and take
// turns at K, U steps at a time, so that a small matrix still fills the chip; their sums, whole numbers, meet
// in LDS.  Lanes of tokens that are not there load nothing.
//
// FUSED: one launch.  Each workgroup quantizes the rows itself into LDS while its first weights fly, which
// costs the chip little at one or a few short rows and saves a launch; at more the rows are quantized once,
// before.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

constexpr int FEW_MAX_T = 32;
constexpr int FEW_WAVES = 8;
constexpr int FEW_FUSED_CODES = 49152;  // bytes of LDS for the rows' codes

template <int RT, int TT, int U, int FUSED, int GATED>
__global__ __launch_bounds__(64 * FEW_WAVES) void k_i8_few(I8Args g) {
    static_assert(!GATED || RT == 2, "a gate tile and an up tile");
    static_assert(!FUSED || TT == 1, "fused for up to 16 tokens");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, q = lane >> 4;
    const int kp = (int)i8_padded(g.k), steps = kp / 64, last = (g.k - 1) & ~15;
    const int t0 = (int)blockIdx.y * 16 * TT;
    const int nt = g.T - t0 < 16 * TT ? g.T - t0 : 16 * TT;
    const int64_t n0 = (int64_t)blockIdx.x * 16 * (GATED ? 1 : RT);
    const int8_t* wr[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        int64_t n = n0 + (GATED ? 0 : 16 * i) + c;
        n = n < g.n_out ? n : g.n_out - 1;
        wr[i] = g.w + (uint64_t)(n + (GATED && i ? g.n_out : 0)) * g.ldw;
    }
    // (a row's pieces past its end: its last one again, against zeros)
    auto load = [&](int s, i8x16 (&to)[U][RT]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            int at = 64 * (s + u) + 16 * q;
            at = at < last ? at : last;
#pragma unroll
            for (int i = 0; i < RT; ++i)
                to[u][i] = __builtin_nontemporal_load(reinterpret_cast<const i8x16*>(wr[i] + at));
        }
    };
    i8x16 cur[U][RT];
    int s = wave * U;
    if (s < steps) load(s, cur);

    const int cs = kp + 16;  // FUSED: the codes' rows in LDS, neighbouring tokens on other banks
    const float* xs = g.xs + t0;
    if constexpr (FUSED) {
        float* fs = reinterpret_cast<float*>(lds);              // [16]
        uint32_t* top = reinterpret_cast<uint32_t*>(lds + 64);  // [16][FEW_WAVES]
        const int es = g.xtype == T_F32 ? 4 : 2;
        auto rows = [&](auto type) {
            constexpr int TY = decltype(type)::value;
            for (int t = 0; t < nt; ++t) {
                const uint8_t* xr = (const uint8_t*)g.x + (uint64_t)(t0 + t) * g.ldx * es;
                uint32_t m = 0;
                float v[8];
                for (int i = threadIdx.x * 8; i < g.k; i += 64 * FEW_WAVES * 8) {
                    i8_load8<TY>(xr, i, g.k, v);
                    m = i8_max8(v, m);
                }
                m = group_max_u32<64>(m);
                if (lane == 0) top[t * FEW_WAVES + wave] = m;
            }
            __syncthreads();
            for (int t = 0; t < nt; ++t) {
                const uint8_t* xr = (const uint8_t*)g.x + (uint64_t)(t0 + t) * g.ldx * es;
                uint32_t m = 0;
#pragma unroll
                for (int w = 0; w < FEW_WAVES; ++w) m = m > top[t * FEW_WAVES + w] ? m : top[t * FEW_WAVES + w];
                const I8Scale sc = i8_scale(m);
                if (threadIdx.x == 0) fs[t] = sc.s;
                float v[8];
                for (int i = threadIdx.x * 8; i < kp; i += 64 * FEW_WAVES * 8) {
                    i8_load8<TY>(xr, i, g.k, v);
                    *reinterpret_cast<uint2*>(lds + 1024 + t * cs + i) = i8_codes8(v, sc.inv);
                }
            }
        };
        if (g.xtype == T_F32)
            rows(std::integral_constant<int, T_F32>{});
        else if (g.xtype == T_F16)
            rows(std::integral_constant<int, T_F16>{});
        else
            rows(std::integral_constant<int, T_BF16>{});
        __syncthreads();
        xs = fs;
    }

    i8x16 acc[RT][TT] = {};
    const int8_t* xr[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) xr[j] = g.xq + (uint64_t)(t0 + 16 * j + c) * kp + 16 * q;
    while (s < steps) {
        const int next = s + U * FEW_WAVES;
        i8x16 nxt[U][RT];
        i8x16 b[U][TT];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < TT; ++j) {
                b[u][j] = i8x16{0, 0, 0, 0};
                if (16 * j + c < nt && s + u < steps) {
                    if constexpr (FUSED)
                        b[u][j] = *reinterpret_cast<const i8x16*>(lds + 1024 + c * cs + 64 * (s + u) + 16 * q);
                    else
                        b[u][j] = *reinterpret_cast<const i8x16*>(xr[j] + 64 * (s + u));
                }
            }
        if (next < steps) load(next, nxt);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < TT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(cur[u][i], b[u][j], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < RT; ++i) cur[u][i] = nxt[u][i];
        s = next;
    }

    // the wavefronts' sums
    i8x16* red = reinterpret_cast<i8x16*>(lds + (FUSED ? 1024 + ((nt * cs + 15) & ~15) : 0));  // [wave][RT TT][64]
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TT; ++j) red[(wave * RT * TT + i * TT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    constexpr int TILES = GATED ? TT : RT * TT;
    if (wave >= TILES) return;
    const int j = GATED ? wave : wave % TT, i = GATED ? 0 : wave / TT;
    i8x16 sum[GATED ? 2 : 1] = {};
#pragma unroll
    for (int m = 0; m < (GATED ? 2 : 1); ++m)
#pragma unroll
        for (int w = 0; w < FEW_WAVES; ++w) sum[m] += red[(w * RT * TT + (i + m) * TT + j) * 64 + lane];
    const int t = 16 * j + c;
    if (t >= nt) return;
    const float sx = xs[t];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t n = n0 + 16 * i + 4 * q + e;
        if (n >= g.n_out) break;
        float v = i8_value(sum[0][e], sx, g.ws[n]);
        if (g.bias) v = v + g.bias[n];
        if constexpr (GATED) {
            float u = i8_value(sum[1][e], sx, g.ws[g.n_out + n]);
            if (g.bias) u = u + g.bias[g.n_out + n];
            v = i8_silu(v) * u;
        }
        i8_store(g.y, g.ytype, (uint64_t)(t0 + t) * g.ldy + n, v);
    }
}

bool i8_few_fits(int T) { return T <= FEW_MAX_T; }

bool i8_few_fused(int rows_w, int k, int T, int gated) {
    (void)rows_w;
    (void)gated;
    return T <= 16 && (uint64_t)T * k <= 16384 && (uint64_t)T * (i8_padded(k) + 16) <= FEW_FUSED_CODES;
}

template <int RT, int TT, int U, int FUSED, int GATED>
static void launch_few(const I8Args& a, hipStream_t stream) {
    const int tiles = a.T < 16 * TT ? a.T : 16 * TT;
    const int lds = FEW_WAVES * RT * TT * 1024 + (FUSED ? 1024 + (tiles * ((int)i8_padded(a.k) + 16) + 15) / 16 * 16 : 0);
    const int per = 16 * (GATED ? 1 : RT);
    static const hipError_t most = hipFuncSetAttribute((const void*)k_i8_few<RT, TT, U, FUSED, GATED>,
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    (void)most;  // a launch that the runtime refuses is reported by the caller
    hipLaunchKernelGGL((k_i8_few<RT, TT, U, FUSED, GATED>), dim3((a.n_out + per - 1) / per, (a.T + 16 * TT - 1) / (16 * TT)),
                       dim3(64 * FEW_WAVES), lds, stream, a);
}

void launch_i8_few(const I8Args& a, hipStream_t stream) {
    if (a.x)
        a.gated ? launch_few<2, 1, 4, 1, 1>(a, stream) : launch_few<1, 1, 8, 1, 0>(a, stream);
    else if (a.T <= 16)
        a.gated ? launch_few<2, 1, 4, 0, 1>(a, stream) : launch_few<1, 1, 8, 0, 0>(a, stream);
    else
        a.gated ? launch_few<2, 2, 4, 0, 1>(a, stream) : launch_few<1, 2, 4, 0, 0>(a, stream);
}

}  // namespace syn
