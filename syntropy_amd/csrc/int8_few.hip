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
// FUSED: up to eight short rows in one launch.  Each workgroup quantizes them into LDS while its first weights
// fly, NW / rows wavefronts a row, a launch less.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

// A fused row's values a wavefront, whole pieces of 8: at most four pieces a lane.
constexpr int FEW_PIECES = 4, FEW_FUSED_WAVES = 8;
constexpr uint64_t FEW_FUSED_MOST = 150000000;
// log2 of the wavefronts a row: eight for one row, four for two, two for three and four, one.
SYN_HD inline int few_share(int rows) { return rows == 1 ? 3 : rows == 2 ? 2 : rows <= 4 ? 1 : 0; }
SYN_HD inline int few_part(int k, int rows) { return (((k + 7) / 8 + (1 << few_share(rows)) - 1) >> few_share(rows)) * 8; }

template <int RT, int TG, int U, int NW, int FUSED, int GATED>  // FUSED: pieces of 8 values a lane, or 0
__global__ __launch_bounds__(64 * NW, TG > 1 || U * RT > 4 ? 4 : 6) void k_i8_few(I8Args g) {
    static_assert(!GATED || RT == 2, "a gate tile and an up tile");
    static_assert(RT * TG <= 4, "the outputs of one wavefront");
    static_assert(!FUSED || TG == 1, "up to eight rows");
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

    // FUSED: the rows' scales, the wavefronts' maxima, the rows' codes (neighbouring rows on other banks)
    float* row_scale = reinterpret_cast<float*>(lds);
    uint8_t* codes = lds + 128;
    const int cs = kp + 16;
    if constexpr (FUSED) {
        uint32_t* top = reinterpret_cast<uint32_t*>(lds + 32);
        auto rows = [&](auto type) {
            constexpr int TY = decltype(type)::value;
            const int share = 1 << few_share(nt), r = wave >> few_share(nt), part = wave & (share - 1);  // uniform
            const int len = few_part(g.k, nt), end = (part + 1) * len < g.k ? (part + 1) * len : g.k;
            const uint8_t* x = (const uint8_t*)g.x + (uint64_t)(t0 + r) * g.ldx * (TY == T_F32 ? 4 : 2);
            float v[FUSED][8];
            uint32_t m = 0;
            if (r < nt) {  // uniform
#pragma unroll
                for (int p = 0; p < FUSED; ++p) {
                    if (512 * p >= len) break;  // uniform
                    i8_load8<TY>(x, part * len + 8 * (lane + 64 * p), end, v[p]);
                }
#pragma unroll
                for (int p = 0; p < FUSED; ++p) {
                    if (512 * p >= len) break;
                    m = i8_max8(v[p], m);
                }
                m = group_max_u32<64>(m);
            }
            if (lane == 0) top[wave] = m;
            __syncthreads();
            if (r < nt) {
                const I8Scale sc = i8_scale(group_max_u32<64>(top[(r << few_share(nt)) + (lane & (share - 1))]));
                if (lane == 0 && part == 0) row_scale[r] = sc.s;
#pragma unroll
                for (int p = 0; p < FUSED; ++p) {
                    if (512 * p >= len) break;
                    const int i = part * len + 8 * (lane + 64 * p);
                    if (8 * (lane + 64 * p) < len && i < kp)
                        *reinterpret_cast<uint2*>(codes + r * cs + i) = i8_codes8(v[p], sc.inv);
                }
                // (zeros from the last part's end to the row's)
                if (part == share - 1)
                    for (int i = share * len + 8 * lane; i < kp; i += 512) *reinterpret_cast<uint2*>(codes + r * cs + i) = uint2{0, 0};
            }
        };
        if (g.xtype == T_F32)
            rows(std::integral_constant<int, T_F32>{});
        else if (g.xtype == T_F16)
            rows(std::integral_constant<int, T_F16>{});
        else
            rows(std::integral_constant<int, T_BF16>{});
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
                    if (c < nt) b = *reinterpret_cast<const i8x16*>(codes + c * cs + I8_LINE * (s + u) + piece);
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
    i8x16* red = reinterpret_cast<i8x16*>(lds + (FUSED ? 128 + nt * cs : 0));  // [wave][RT][TG][64]
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
    const float sx = FUSED ? row_scale[t] : g.xs[t0 + t];
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

// Up to 8 tokens; up to 16 over matrices that have too few tiles for the chip (4096 x 4096 at 16 tokens 7.5 us
// against 9.5 in tiles, 6144 x 4096 11.0 against 7.9).
bool i8_few_fits(int rows_w, int T) { return T <= 8 || (T <= 16 && rows_w <= 5120); }

// One row, or as many as take each workgroup no longer than a launch (a value costs a workgroup's wavefronts
// about eight operations), where the wavefronts' registers hold them.  4096 x 4096 at one row 6.7 us against 8.2
// with the row quantized in a launch before.
bool i8_few_fused(int rows_w, int k, int T) {
    if (T < 1 || T > 8 || few_part(k, T) > 512 * FEW_PIECES) return false;
    return T == 1 || (uint64_t)rows_w * (uint64_t)T * (uint64_t)k <= FEW_FUSED_MOST;
}

template <int RT, int TG, int U, int NW, int FUSED, int GATED>
static void launch_few(const I8Args& a, hipStream_t stream) {
    const int lds = NW * RT * TG * 1024 + (FUSED ? 128 + a.T * ((int)i8_padded(a.k) + 16) : 0);
    const int per = 8 * (GATED ? 1 : RT);
    static std::atomic<uint64_t> said{0};
    i8_allow_lds((const void*)k_i8_few<RT, TG, U, NW, FUSED, GATED>, 160 * 1024, said);
    hipLaunchKernelGGL((k_i8_few<RT, TG, U, NW, FUSED, GATED>), dim3((a.n_out + per - 1) / per, (a.T + 8 * TG - 1) / (8 * TG)),
                       dim3(64 * NW), lds, stream, a);
}

template <int RT, int GATED>
static void launch_rows(const I8Args& a, hipStream_t stream) {
    if (a.T > 8)
        launch_few<2, 2, 2, 8, 0, GATED>(a, stream);
    else if (!a.x)
        launch_few<RT, 1, 2, 8, 0, GATED>(a, stream);
    else if (few_part(a.k, a.T) <= 512)  // (with the registers of more, fewer workgroups a CU)
        launch_few<RT, 1, 2, FEW_FUSED_WAVES, 1, GATED>(a, stream);
    else
        launch_few<RT, 1, 2, FEW_FUSED_WAVES, FEW_PIECES, GATED>(a, stream);
}

// Rows of weights a workgroup: 8 for one or two tokens (14336 x 4096 at 1 token 12.5 us against 13.3 for 16, at 2
// 14.4 against 15.0), else 16, which share the tokens' codes (at 8 tokens 17.7 against 19.0).  Two lines a
// turn: with four the registers leave too few wavefronts (1 token, 8 rows, 15.3).
static void launch_some(const I8Args& a, hipStream_t stream) {
    if (a.gated)
        launch_rows<2, 1>(a, stream);
    else if (a.T <= 2)
        launch_rows<1, 0>(a, stream);
    else
        launch_rows<2, 0>(a, stream);
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
