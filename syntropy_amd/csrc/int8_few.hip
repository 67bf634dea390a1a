// The int8 product at few tokens (one to 16): bound by reading the weights once from HBM.
//
// v_mfma_i32_16x16x64_i8 multiplies 16 rows by 16 columns over 64 values, four lanes a row of 16 codes each.
// Its rows are taken as 8 weight rows x the two halves of a 128-byte line and its columns as 8 tokens x the
// same halves: where a row's half is a column's, the product is one that is wanted (the other half of the
// matrix cores' work, which cost nothing here, is not looked at).  So a lane loads 16 codes of a weight row
// straight to the registers that the instruction reads, and an instruction loads whole 128-byte lines of 8
// rows: 14336 x 4096 read that way takes 12.2 us, 64 bytes of each of 16 rows 15.8, a row 11.9.  No other
// wavefront reads those codes, so LDS would only be a detour.
// The eight wavefronts of a workgroup share 8 RT rows and take turns at K, U lines at a time, so that a small
// matrix still fills the chip, two turns in flight; their sums, whole numbers, meet in LDS.  A wavefront keeps to
// few registers, so that most matrices are asked for whole at once.  Lanes of tokens that are not there load
// nothing.
//
// The tokens' codes of a turn are loaded with its weights: loads return in order, so that codes asked for when
// they are needed would wait for the next turn's weights too.
//
// FUSED: one row in one launch.  Each workgroup quantizes it into LDS while its first weights fly, a launch
// less.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

constexpr int FEW_MAX_T = 16;

template <int RT, int TG, int U, int NW, int FUSED, int GATED>
__global__ __launch_bounds__(64 * NW, TG > 1 || U * RT > 4 ? 4 : 6) void k_i8_few(I8Args g) {
    static_assert(!GATED || RT == 2, "a gate tile and an up tile");
    static_assert(RT * TG <= 4, "the outputs of one wavefront");
    static_assert(!FUSED || TG == 1, "one row");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 7;                                        // weight row, and token, of 8
    const int piece = 16 * (4 * ((lane >> 3) & 1) + (lane >> 4));  // of a line
    const int kp = (int)i8_padded(g.k), lines = kp / I8_LINE, last = (g.k - 1) & ~15;
    const int t0 = (int)blockIdx.y * 8 * TG;
    const int nt = g.T - t0 < 8 * TG ? g.T - t0 : 8 * TG;
    const int64_t n0 = (int64_t)blockIdx.x * 8 * (GATED ? 1 : RT);
    const int8_t* wr[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        int64_t n = n0 + (GATED ? 0 : 8 * i) + c;
        n = n < g.n_out ? n : g.n_out - 1;
        wr[i] = g.w + (uint64_t)(n + (GATED && i ? g.n_out : 0)) * g.ldw;
    }
    const int8_t* xr = FUSED ? nullptr : g.xq + (uint64_t)(t0 + c) * kp + piece;
    constexpr int TURN = U * NW;  // lines
    struct Turn {
        i8x16 w[U][RT], x[FUSED ? 1 : U][TG];
    };
    auto load = [&](int s, Turn& to) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= lines) break;  // uniform
            int at = I8_LINE * (s + u) + piece;
            at = at < last ? at : last;  // a row's pieces past its end: its last one again, against zeros
#pragma unroll
            for (int i = 0; i < RT; ++i)
                to.w[u][i] = __builtin_nontemporal_load(reinterpret_cast<const i8x16*>(wr[i] + at));
            if constexpr (!FUSED) {
#pragma unroll
                for (int j = 0; j < TG; ++j) {
                    to.x[u][j] = i8x16{0, 0, 0, 0};
                    if (8 * j + c < nt)
                        to.x[u][j] = *reinterpret_cast<const i8x16*>(xr + (uint64_t)(8 * j) * kp + I8_LINE * (s + u));
                }
            }
        }
    };
    Turn cur, nxt;
    int s = wave * U;
    load(s, cur);
    load(s + TURN, nxt);

    float* row_scale = reinterpret_cast<float*>(lds);  // FUSED: the row's scale, the wavefronts' maxima, its codes
    uint8_t* codes = lds + 128;
    if constexpr (FUSED) {
        uint32_t* top = reinterpret_cast<uint32_t*>(lds + 16);
        auto row = [&](auto type) {
            constexpr int TY = decltype(type)::value;
            const uint8_t* x = (const uint8_t*)g.x + (uint64_t)t0 * g.ldx * (TY == T_F32 ? 4 : 2);
            float v[2][8];  // i8_few_fused: a row is at most two pieces of 8 a thread
            uint32_t m = 0;
#pragma unroll
            for (int p = 0; p < 2; ++p) i8_load8<TY>(x, 8 * ((int)threadIdx.x + 64 * NW * p), g.k, v[p]);
#pragma unroll
            for (int p = 0; p < 2; ++p) m = i8_max8(v[p], m);
            m = group_max_u32<64>(m);
            if (lane == 0) top[wave] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) m = m > top[w] ? m : top[w];
            const I8Scale sc = i8_scale(m);
            if (threadIdx.x == 0) *row_scale = sc.s;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int i = 8 * ((int)threadIdx.x + 64 * NW * p);
                if (i < kp) *reinterpret_cast<uint2*>(codes + i) = i8_codes8(v[p], sc.inv);
            }
        };
        if (g.xtype == T_F32)
            row(std::integral_constant<int, T_F32>{});
        else if (g.xtype == T_F16)
            row(std::integral_constant<int, T_F16>{});
        else
            row(std::integral_constant<int, T_BF16>{});
        __syncthreads();
    }

    i8x16 acc[RT][TG] = {};
    auto product = [&](int s, const Turn& o) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= lines) break;  // uniform
#pragma unroll
            for (int j = 0; j < TG; ++j) {
                i8x16 b;
                if constexpr (FUSED) {
                    b = i8x16{0, 0, 0, 0};
                    if (c == 0) b = *reinterpret_cast<const i8x16*>(codes + I8_LINE * (s + u) + piece);
                } else {
                    b = o.x[u][j];
                }
#pragma unroll
                for (int i = 0; i < RT; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.w[u][i], b, acc[i][j], 0, 0, 0);
            }
        }
    };
    while (s < lines) {  // uniform
        product(s, cur);
        load(s + 2 * TURN, cur);
        s += TURN;
        product(s, nxt);
        load(s + 2 * TURN, nxt);
        s += TURN;
    }

    // The wavefronts' sums.  Lane l holds columns l & 15, rows 4 (l >> 4) .. + 3 of 16: those of the first half
    // by the first (lanes 0..7 and 16..23) and of the second by the second (40..47 and 56..63).
    i8x16* red = reinterpret_cast<i8x16*>(lds + (FUSED ? 128 + kp : 0));  // [wave][RT][TG][64]
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < TG; ++j) red[((wave * RT + i) * TG + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    if (wave != 0) return;
    // lane: tile l / 16 of the (RT or, gated, 1) x TG, rows 4 (l / 8 & 1) .. + 3, token l & 7
    const int tile = lane >> 4, half = (lane >> 3) & 1;
    if (tile >= (GATED ? 1 : RT) * TG) return;
    const int i = GATED ? 0 : tile / TG, j = GATED ? tile : tile % TG, t = 8 * j + c;
    i8x16 sum[GATED ? 2 : 1] = {};
#pragma unroll
    for (int m = 0; m < (GATED ? 2 : 1); ++m)
#pragma unroll 4
        for (int w = 0; w < NW; ++w) {
            const i8x16* r = red + ((w * RT + i + m) * TG + j) * 64;
            sum[m] += r[16 * half + c] + r[16 * half + 40 + c];
        }
    if (t >= nt) return;
    const float sx = FUSED ? *row_scale : g.xs[t0 + t];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t n = n0 + 8 * i + 4 * half + e;
        if (n >= g.n_out) break;
        float v = i8_value(sum[0][e], sx, g.ws[n]);
        if (g.bias) v = v + g.bias[n];
        if constexpr (GATED) {
            float u = i8_value(sum[GATED ? 1 : 0][e], sx, g.ws[g.n_out + n]);
            if (g.bias) u = u + g.bias[g.n_out + n];
            v = i8_silu(v) * u;
        }
        i8_store(g.y, g.ytype, (uint64_t)(t0 + t) * g.ldy + n, v);
    }
}

bool i8_few_fits(int T) { return T <= FEW_MAX_T; }

// One row of at most two pieces of 8 values a thread of the largest workgroup (4096 x 4096: 6.7 against 8.2 us
// with the row quantized in a launch before).
bool i8_few_fused(int k, int T) { return T == 1 && k <= 16384; }

template <int RT, int TG, int U, int NW, int FUSED, int GATED>
static void launch_few(const I8Args& a, hipStream_t stream) {
    const int lds = NW * RT * TG * 1024 + (FUSED ? 128 + (int)i8_padded(a.k) : 0);
    const int per = 8 * (GATED ? 1 : RT);
    static const hipError_t most = hipFuncSetAttribute((const void*)k_i8_few<RT, TG, U, NW, FUSED, GATED>,
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    (void)most;  // a launch that the runtime refuses is reported by the caller
    hipLaunchKernelGGL((k_i8_few<RT, TG, U, NW, FUSED, GATED>), dim3((a.n_out + per - 1) / per, (a.T + 8 * TG - 1) / (8 * TG)),
                       dim3(64 * NW), lds, stream, a);
}

// Rows of weights a workgroup: 8 for one or two tokens (14336 x 4096 at 1 token 12.5 us against 13.3 for 16, at 2
// 14.4 against 15.0), else 16, which share the tokens' codes (at 8 tokens 17.7 against 19.0).  Two lines a
// turn: with four the registers leave too few wavefronts (1 token, 8 rows, 15.3).  Long fused rows on 16
// wavefronts, for the quantization's sake.
static void launch_some(const I8Args& a, hipStream_t stream) {
    const bool wide = a.x && a.k > 8192;
    if (a.T > 8)
        a.gated ? launch_few<2, 2, 2, 8, 0, 1>(a, stream) : launch_few<2, 2, 2, 8, 0, 0>(a, stream);
    else if (a.gated && a.x)
        wide ? launch_few<2, 1, 2, 16, 1, 1>(a, stream) : launch_few<2, 1, 2, 8, 1, 1>(a, stream);
    else if (a.gated)
        launch_few<2, 1, 2, 8, 0, 1>(a, stream);
    else if (a.x)
        wide ? launch_few<1, 1, 2, 16, 1, 0>(a, stream) : launch_few<1, 1, 2, 8, 1, 0>(a, stream);
    else if (a.T <= 2)
        launch_few<1, 1, 2, 8, 0, 0>(a, stream);
    else
        launch_few<2, 1, 2, 8, 0, 0>(a, stream);
}

// (any number of tokens, for weight rows that a tile's offsets do not reach: as many a launch as a grid holds)
void launch_i8_few(const I8Args& a, hipStream_t stream) {
    constexpr int MOST = 1 << 19;
    for (int t = 0; t < a.T; t += MOST) {
        I8Args g = a;
        g.T = a.T - t < MOST ? a.T - t : MOST;
        g.xq = a.xq + (uint64_t)t * i8_padded(a.k);
        g.xs = a.xs + t;
        g.y = (uint8_t*)a.y + (uint64_t)t * a.ldy * (a.ytype == T_F32 ? 4 : 2);
        launch_some(g, stream);
    }
}

}  // namespace syn
