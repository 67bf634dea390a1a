// The int8 product at many tokens on v_mfma_i32_32x32x32_i8.
//
// A workgroup of WM x WN wavefronts takes a tile of 32 MT WM tokens x 32 NT WN weight rows, 128 values (a line)
// of every row a stage; each stage's lines are copied into LDS by global_load_lds one stage ahead.  Piece p
// (16 bytes) of line r lies at p ^ (r & 7), so that eight neighbouring lines' same pieces are on eight
// different bank groups.  The tokens are the instruction's A rows, the weight rows its columns: a lane holds
// one output column's 16 tokens a tile, and 32 lanes write 32 neighbouring outputs.
// GATED: a wavefront's columns are half gate rows, half the same up rows, so that it holds both values.
// Where the tiles are too few to fill the chip, K is split over gridDim.z workgroups: whole-number partial
// sums to the workspace, added by k_i8_fold.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

constexpr int GEMM_STAGES = 2;

template <int WM, int WN, int MT, int NT>
struct I8Tile {
    static constexpr int NW = WM * WN, BM = 32 * MT * WM, BN = 32 * NT * WN;
    static constexpr int XI = BM / 8, WI = BN / 8;  // copy instructions a stage, of 8 lines each
    static constexpr int XPW = (XI + NW - 1) / NW, WPW = (WI + NW - 1) / NW;
    static constexpr int STAGE = (BM + BN) * I8_LINE;
    static constexpr int LDS = GEMM_STAGES * STAGE;
    static_assert(XI % NW == 0 && WI % NW == 0, "every wavefront copies as many lines");
};

template <int WM, int WN, int MT, int NT, int GATED>
__global__ __launch_bounds__(64 * WM * WN, 1) void k_i8_gemm(I8Args g, int tiles_n, int tiles_m) {
    using C = I8Tile<WM, WN, MT, NT>;
    static_assert(!GATED || NT % 2 == 0, "gate columns and up columns");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int c = lane & 31, h = lane >> 5;
    const int tm = (int)blockIdx.x % tiles_m, tn = (int)blockIdx.x / tiles_m;
    const int t0 = tm * C::BM;
    const int n0 = tn * (GATED ? C::BN / 2 : C::BN);
    const int kp = (int)i8_padded(g.k), stages = kp / I8_LINE;
    const int z = (int)blockIdx.z;
    const int s0 = (int)((int64_t)stages * z / g.splits), s1 = (int)((int64_t)stages * (z + 1) / g.splits);

    // this wavefront's copies: lines 8 (wave + NW i) .. + 7, lane l line l / 8, piece l % 8 of LDS
    const uint32_t piece = 16u * (uint32_t)((lane & 7) ^ (lane >> 3));
    uint32_t xo[C::XPW], wo[C::WPW];
    const int8_t* wb[GATED ? 2 : 1];
    const int8_t* xb = g.xq + (uint64_t)t0 * kp;
    wb[0] = g.w + (uint64_t)n0 * g.ldw;
    if constexpr (GATED) wb[1] = wb[0] + (uint64_t)g.n_out * g.ldw;
#pragma unroll
    for (int i = 0; i < C::XPW; ++i) {
        int t = 8 * (wave + C::NW * i) + (lane >> 3);
        t = t0 + t < g.T ? t : g.T - 1 - t0;
        xo[i] = (uint32_t)t * (uint32_t)kp + piece;
    }
    constexpr int WC = 32 * NT;  // a wavefront's columns
    auto up_half = [&](int i) { return GATED && 8 * (wave + C::NW * i) % WC >= WC / 2; };  // uniform
#pragma unroll
    for (int i = 0; i < C::WPW; ++i) {
        const int l = 8 * (wave + C::NW * i) + (lane >> 3);
        int n = GATED ? l / WC * (WC / 2) + l % (WC / 2) : l;
        n = n0 + n < g.n_out ? n : g.n_out - 1 - n0;
        wo[i] = (uint32_t)n * (uint32_t)g.ldw + piece;
    }
    // in the last stage a weight row's pieces past its end: its last one again, against zeros
    const uint32_t lastp = (uint32_t)(g.k - 1) & ~15u;
    const uint32_t endp = (uint32_t)I8_LINE * (uint32_t)(stages - 1) + piece;
    const uint32_t end_adj = (endp < lastp ? endp : lastp) - piece;
    const uint32_t ring = lds_addr(lds);
    auto copy = [&](int s) {
        const uint32_t to = ring + (uint32_t)((s - s0) % GEMM_STAGES) * C::STAGE;
#pragma unroll
        for (int i = 0; i < C::XPW; ++i)
            lds_dma16(xo[i], xb + (uint64_t)s * I8_LINE, to + 1024u * (uint32_t)(wave + C::NW * i));
        const uint32_t tw = to + C::BM * I8_LINE;
        if (s != stages - 1) {
#pragma unroll
            for (int i = 0; i < C::WPW; ++i)
                lds_dma16(wo[i], wb[up_half(i)] + (uint64_t)s * I8_LINE, tw + 1024u * (uint32_t)(wave + C::NW * i));
        } else {
#pragma unroll
            for (int i = 0; i < C::WPW; ++i)
                lds_dma16(wo[i] + end_adj, wb[up_half(i)], tw + 1024u * (uint32_t)(wave + C::NW * i));
        }
    };

    i32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x16{};

    if (s0 < s1) copy(s0);
    for (int s = s0; s < s1; ++s) {
        wait_vm<0>();
        lds_barrier();
        if (s + 1 < s1) copy(s + 1);
        const uint8_t* st = lds + (uint32_t)((s - s0) % GEMM_STAGES) * C::STAGE;
        const uint8_t* xl = st + (wm * 32 * MT + c) * I8_LINE;
        const uint8_t* wl = st + C::BM * I8_LINE + (wn * 32 * NT + c) * I8_LINE;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int p = 16 * ((2 * kk + h) ^ (c & 7));
            i8x16 a[MT], b[NT];
#pragma unroll
            for (int i = 0; i < MT; ++i) a[i] = *reinterpret_cast<const i8x16*>(xl + i * 32 * I8_LINE + p);
#pragma unroll
            for (int j = 0; j < NT; ++j) b[j] = *reinterpret_cast<const i8x16*>(wl + j * 32 * I8_LINE + p);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
        }
    }

    // lane: column c of each tile of 32, tokens 8 (e / 4) + 4 h + e % 4
    const uint64_t rows_w = (uint64_t)g.n_out * (GATED ? 2 : 1);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int tb = t0 + (wm * MT + i) * 32 + 4 * h;
        if (g.splits > 1) {
            int* part = g.partial + (uint64_t)z * g.T * rows_w;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int half = GATED && j >= NT / 2;
                const int n = n0 + (GATED ? wn * (WC / 2) + (j % (NT / 2)) * 32 : wn * WC + j * 32) + c;
                if (n >= g.n_out) continue;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int t = tb + 8 * (e / 4) + e % 4;
                    if (t < g.T) part[(uint64_t)t * rows_w + (uint64_t)half * g.n_out + n] = acc[i][j][e];
                }
            }
            continue;
        }
        float sx[16];
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4 v = *reinterpret_cast<const float4*>(g.xs + tb + 2 * e);
            sx[e] = v.x, sx[e + 1] = v.y, sx[e + 2] = v.z, sx[e + 3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < (GATED ? NT / 2 : NT); ++j) {
            const int n = n0 + (GATED ? wn * (WC / 2) : wn * WC) + j * 32 + c;
            if (n >= g.n_out) continue;
            const float sw = g.ws[n], bw = g.bias ? g.bias[n] : 0.0f;
            float su = 0.0f, bu = 0.0f;
            if constexpr (GATED) su = g.ws[g.n_out + n], bu = g.bias ? g.bias[g.n_out + n] : 0.0f;
            auto out = [&](int e) {
                float v = i8_value(acc[i][j][e], sx[e], sw);
                if (g.bias) v = v + bw;
                if constexpr (GATED) {
                    float u = i8_value(acc[i][j + (GATED ? NT / 2 : 0)][e], sx[e], su);
                    if (g.bias) u = u + bu;
                    v = ref_silu(v) * u;
                }
                return v;
            };
            const uint64_t at = (uint64_t)tb * g.ldy + n;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int d = 8 * (e / 4) + e % 4;
                if (tb + d < g.T) i8_store(g.y, g.ytype, at + (uint64_t)d * g.ldy, out(e));
            }
        }
    }
}

// The tiles, tokens x weight rows.
enum : int { TILE_256x256 = 0, TILE_128x128 = 1, TILE_64x128 = 2, TILE_64x64 = 3, TILES = 4 };
static const int TILE_M[TILES] = {256, 128, 64, 64}, TILE_N[TILES] = {256, 128, 128, 64};

I8Pick i8_gemm_pick(int rows_w, int k, int T, int gated) {
    (void)gated;
    I8Pick p{TILE_64x64, 1};
    for (int i = 0; i < TILES; ++i) {
        p.tile = i;
        const int64_t tiles = (int64_t)((T + TILE_M[i] - 1) / TILE_M[i]) * ((rows_w + TILE_N[i] - 1) / TILE_N[i]);
        if (tiles >= 200) return p;
    }
    const int64_t tiles = (int64_t)((T + 63) / 64) * ((rows_w + 63) / 64);
    const int stages = (int)(i8_padded(k) / I8_LINE);
    int s = (int)(256 / tiles);
    if (s > stages / 4) s = stages / 4;
    p.splits = s < 1 ? 1 : s;
    return p;
}

bool i8_gemm_reaches(int tile, const I8Args& a) { return (uint64_t)TILE_N[tile] * a.ldw < (1ull << 31); }

template <int WM, int WN, int MT, int NT, int GATED>
static void launch_tile(const I8Args& a, hipStream_t stream) {
    using C = I8Tile<WM, WN, MT, NT>;
    const int bn = GATED ? C::BN / 2 : C::BN;
    const int tn = (a.n_out + bn - 1) / bn, tm = (a.T + C::BM - 1) / C::BM;
    static const hipError_t lds = hipFuncSetAttribute((const void*)k_i8_gemm<WM, WN, MT, NT, GATED>,
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
    (void)lds;  // a launch that the runtime refuses is reported by the caller
    hipLaunchKernelGGL((k_i8_gemm<WM, WN, MT, NT, GATED>), dim3((uint32_t)tn * (uint32_t)tm, 1, a.splits), dim3(64 * C::NW),
                       C::LDS, stream, a, tn, tm);
}
template <int WM, int WN, int MT, int NT>
static void launch_tile(const I8Args& a, hipStream_t stream) {
    a.gated ? launch_tile<WM, WN, MT, NT, 1>(a, stream) : launch_tile<WM, WN, MT, NT, 0>(a, stream);
}

void launch_i8_gemm(int tile, const I8Args& a, hipStream_t stream) {
    switch (tile) {
    case TILE_256x256: launch_tile<2, 2, 4, 4>(a, stream); break;
    case TILE_128x128: launch_tile<2, 2, 2, 2>(a, stream); break;
    case TILE_64x128: launch_tile<2, 2, 1, 2>(a, stream); break;
    default: launch_tile<2, 1, 1, 2>(a, stream); break;
    }
}

}  // namespace syn
