// The int8 product at many tokens on v_mfma_i32_32x32x32_i8.
//
// A workgroup of WM x WN wavefronts takes a tile of 32 MT WM weight rows x 32 NT WN tokens, a wavefront 32 MT x
// 32 NT of it, 64 values of every row a stage.  The stages' lines are copied into a ring of four in LDS by
// global_load_lds, three stages ahead.  Piece p (16 bytes) of line r lies at p ^ (r / 2 & 3), so that eight
// neighbouring lines' same pieces are on eight different bank groups.
// Each half stage's operands are read into registers during the half stage before, the first half of the next
// stage's behind the stage's one barrier, and all of it (products, reads, copies) is written in the order in
// which it is to be issued and held there: a large tile leaves one wavefront a SIMD, whose matrix products
// nothing else covers.  Left to itself the compiler reads each operand right before its product.
// The weight rows are the instruction's A rows, the tokens its columns: a lane holds four neighbouring outputs
// of a token at a time, which go through LDS to whole 16-byte pieces of y's rows.
// GATED: a wavefront's rows are half gate rows, half the same up rows, so that it holds both values.
// Where the tiles are too few to fill the chip, K is split over gridDim.z workgroups: whole-number partial
// sums to the workspace, added by k_i8_fold.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

constexpr int GEMM_RING = 4;   // stages in LDS
constexpr int GEMM_BK = 64;    // values a stage

template <int N, class F, int I = 0>
SYN_DEV void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<N, F, I + 1>(static_cast<F&&>(f));
    }
}

template <int WM, int WN, int MT, int NT>
struct I8Tile {
    static constexpr int NW = WM * WN, BM = 32 * MT * WM, BN = 32 * NT * WN;
    static constexpr int WPW = BM / 16 / NW, XPW = BN / 16 / NW;  // a wavefront's copies a stage, 16 lines each
    static constexpr int CPW = WPW + XPW;
    static constexpr int STAGE = (BM + BN) * GEMM_BK;
    // a wavefront's outputs of 32 tokens on their way out, its rows' scales and biases
    static constexpr int OUT = 32 * (32 * MT * 4 + 16) + 32 * MT * 8;
    static constexpr int LDS = GEMM_RING * STAGE > NW * OUT ? GEMM_RING * STAGE : NW * OUT;
    static_assert(BM % (16 * NW) == 0 && BN % (16 * NW) == 0, "every wavefront copies as many lines");
    static constexpr int C0 = CPW / 2;                   // of them issued in a stage's first half
    static_assert(CPW * 2 < 64, "vmcnt");
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <int WM, int WN, int MT, int NT, int GATED, int TY>
__global__ __launch_bounds__(64 * WM * WN, MT* NT >= 16 ? 1 : 2) void k_i8_gemm(I8Args g, int tiles_w, int tiles_t) {
    using C = I8Tile<WM, WN, MT, NT>;
    static_assert(!GATED || MT % 2 == 0, "gate rows and up rows");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
    const int c = lane & 31, h = lane >> 5;
    int tw, tt;
    i8_tile_of((int)blockIdx.x, tiles_w, tiles_t, tw, tt);
    const int t0 = tt * C::BN;
    const int n0 = tw * (GATED ? C::BM / 2 : C::BM);
    const int kp = (int)i8_padded(g.k), stages = kp / GEMM_BK;
    const int z = (int)blockIdx.z;
    const int s0 = (int)((int64_t)stages * z / g.splits), s1 = (int)((int64_t)stages * (z + 1) / g.splits);

    // this wavefront's copies: lines 16 (wave + NW i) .. + 15, lane l line l / 4, place l % 4 of it
    const uint32_t piece = 16u * (uint32_t)((lane & 3) ^ ((lane >> 3) & 3));
    uint32_t wo[C::WPW], xo[C::XPW];
    const int8_t* wb[GATED ? 2 : 1];
    const int8_t* xb = g.xq + (uint64_t)t0 * kp;
    wb[0] = g.w + (uint64_t)n0 * g.ldw;
    if constexpr (GATED) wb[1] = wb[0] + (uint64_t)g.n_out * g.ldw;
    constexpr int WR = 32 * MT;  // a wavefront's rows
    auto up_half = [&](int i) { return GATED && 16 * (wave + C::NW * i) % WR >= WR / 2; };  // uniform
#pragma unroll
    for (int i = 0; i < C::WPW; ++i) {
        const int l = 16 * (wave + C::NW * i) + (lane >> 2);
        int n = GATED ? l / WR * (WR / 2) + l % (WR / 2) : l;
        n = n0 + n < g.n_out ? n : g.n_out - 1 - n0;
        wo[i] = (uint32_t)n * (uint32_t)g.ldw + piece;
    }
#pragma unroll
    for (int i = 0; i < C::XPW; ++i) {
        int t = 16 * (wave + C::NW * i) + (lane >> 2);
        t = t0 + t < g.T ? t : g.T - 1 - t0;
        xo[i] = (uint32_t)t * (uint32_t)kp + piece;
    }
    const uint32_t ring = lds_addr(lds);
    const int whole = g.k / GEMM_BK;                       // stages that every weight row fills
    const uint32_t lastp = (uint32_t)(g.k - 1) & ~15u;     // a row's last piece
    // What the copies of stage s share: the ring's place for it, and where it lies in a row.  Past a weight
    // row's end its last piece again, against zeros.  Past the part's last stage that one again, into places
    // that are read by nothing that counts: the loop has one form.
    struct Where {
        uint32_t to, adj;
        uint64_t w, x;
    };
    auto where = [&](int s) {
        Where v;
        v.to = ring + (uint32_t)(s & (GEMM_RING - 1)) * C::STAGE;
        s = s < s1 ? s : s1 - 1;
        const uint32_t p = (uint32_t)s * GEMM_BK + piece;
        v.adj = s < whole ? 0u : (p < lastp ? p : lastp) - piece;
        v.w = s < whole ? (uint64_t)s * GEMM_BK : 0u;
        v.x = (uint64_t)s * GEMM_BK;
        return v;
    };
    // copy i of a stage: the weight rows' first, then the tokens'
    auto copy = [&](const Where& v, int i) {
        if (i < C::WPW) {
            const int j = i < C::WPW ? i : 0;
            lds_dma16(wo[j] + v.adj, wb[up_half(j)] + v.w, v.to + 1024u * (uint32_t)(wave + C::NW * j));
        } else {
            const int j = i - C::WPW;
            lds_dma16(xo[j], xb + v.x, v.to + C::BM * GEMM_BK + 1024u * (uint32_t)(wave + C::NW * j));
        }
    };

    i32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x16{};

    i8x16 a[2][MT], b[2][NT];
    const int place = 16 * (h ^ ((c >> 1) & 3));  // of piece h; piece 2 + h lies at place ^ 32
    const uint8_t* al = lds + (wm * WR + c) * GEMM_BK;
    const uint8_t* bl = lds + C::BM * GEMM_BK + (wn * 32 * NT + c) * GEMM_BK;
    // operand r of half kk of stage s into buffer kk
    auto read = [&](int s, int kk, int r) {
        const int off = (s & (GEMM_RING - 1)) * C::STAGE + (place ^ (32 * kk));
        if (r < MT)
            a[kk][r < MT ? r : 0] = *reinterpret_cast<const i8x16*>(al + off + (r < MT ? r : 0) * 32 * GEMM_BK);
        else
            b[kk][r - MT] = *reinterpret_cast<const i8x16*>(bl + off + (r - MT) * 32 * GEMM_BK);
    };
    // the products of half kk, the reads of the other buffer's half and half of a stage's copies among them
    auto half = [&](auto kkc, int rs, int cs) {
        constexpr int kk = decltype(kkc)::value;
        const Where v = where(cs);
        constexpr int M = MT * NT, R = MT + NT, first = kk ? C::C0 : 0, CP = kk ? C::CPW - C::C0 : C::C0;
        static_for<M>([&](auto mc) {
            constexpr int m = decltype(mc)::value, i = m / NT, j = m % NT;
            acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[kk][i], b[kk][j], acc[i][j], 0, 0, 0);
            // reads in the first half of the products (one or more a product), copies in the second
            constexpr int H = M / 2;
            constexpr int r0 = m < H ? m * R / H : R, r1 = m < H ? (m + 1) * R / H : R;
            if constexpr (r1 > r0) static_for<r1 - r0>([&](auto rc) { read(rs, 1 - kk, r0 + decltype(rc)::value); });
            constexpr int c0 = m >= H ? (m - H) * CP / (M - H) : 0, c1 = m >= H ? (m - H + 1) * CP / (M - H) : 0;
            if constexpr (c1 > c0) static_for<c1 - c0>([&](auto cc) { copy(v, first + c0 + decltype(cc)::value); });
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    static_for<GEMM_RING - 1>([&](auto sc) {
        const Where v = where(s0 + decltype(sc)::value);
        static_for<C::CPW>([&](auto i) { copy(v, decltype(i)::value); });
    });
    wait_vm<(GEMM_RING - 2) * C::CPW>();
    lds_barrier();
    static_for<MT + NT>([&](auto r) { read(s0, 0, decltype(r)::value); });
    for (int s = s0; s < s1; ++s) {
        half(std::integral_constant<int, 0>{}, s, s + GEMM_RING - 1);
        wait_vm<(GEMM_RING - 3) * C::CPW + C::C0>();  // stage s + 1 is there
        lds_barrier();
        half(std::integral_constant<int, 1>{}, s + 1, s + GEMM_RING - 1);
    }
    wait_vm<0>();
    lds_barrier();  // the ring is free

    // lane: token c of each tile of 32, rows 8 e4 + 4 h + 0..3
    uint8_t* mine = lds + wave * C::OUT;
    {  // TY: an output type, or -1: the sums of a part of K
        constexpr int ES = TY == T_F32 || TY < 0 ? 4 : 2;
        constexpr int OC = GATED && TY >= 0 ? WR / 2 : WR;  // outputs a token
        constexpr int PITCH = OC * ES + 16, PIECES = OC * ES / 16, PER = 16 / ES;
        const uint64_t rows_w = (uint64_t)g.n_out * (GATED ? 2 : 1);
        uint8_t* out = TY < 0 ? (uint8_t*)(g.partial + (uint64_t)z * g.T * rows_w) : (uint8_t*)g.y;
        const uint64_t pitch = (TY < 0 ? rows_w : g.ldy) * ES;
        float* sw = reinterpret_cast<float*>(mine + 32 * (WR * 4 + 16));  // [WR], then the biases
        if constexpr (TY >= 0) {
            for (int r = lane; r < WR; r += 64) {
                int n = n0 + (GATED ? wm * (WR / 2) + r % (WR / 2) : wm * WR + r);
                n = (n < g.n_out ? n : g.n_out - 1) + (GATED && r >= WR / 2 ? g.n_out : 0);
                sw[r] = g.ws[n];
                sw[WR + r] = g.bias ? g.bias[n] : 0.0f;
            }
            wave_lds_sync();
        }
        static_for<NT>([&](auto jc) {
            constexpr int j = decltype(jc)::value;
            const int tb = t0 + (wn * NT + j) * 32;
            const float sx = g.xs[tb + c];
            static_for<OC / 32>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int o = i * 32 + 8 * e4 + 4 * h;  // of the wavefront's outputs
                    uint8_t* to = mine + c * PITCH + o * ES;
                    if constexpr (TY < 0) {
                        *reinterpret_cast<i8x16*>(to) = i8x16{acc[i][j][4 * e4], acc[i][j][4 * e4 + 1], acc[i][j][4 * e4 + 2],
                                                              acc[i][j][4 * e4 + 3]};
                    } else {
                        float v[4];
                        const float4 sv = *reinterpret_cast<const float4*>(sw + o), bv = *reinterpret_cast<const float4*>(sw + WR + o);
                        const float sg[4] = {sv.x, sv.y, sv.z, sv.w}, bg[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            v[e] = i8_value(acc[i][j][4 * e4 + e], sx, sg[e]);
                            if (g.bias) v[e] = v[e] + bg[e];
                        }
                        if constexpr (GATED) {
                            const float4 su = *reinterpret_cast<const float4*>(sw + WR / 2 + o);
                            const float4 bu = *reinterpret_cast<const float4*>(sw + WR + WR / 2 + o);
                            const float s2[4] = {su.x, su.y, su.z, su.w}, b2[4] = {bu.x, bu.y, bu.z, bu.w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float u = i8_value(acc[i + (GATED ? MT / 2 : 0)][j][4 * e4 + e], sx, s2[e]);
                                if (g.bias) u = u + b2[e];
                                v[e] = i8_silu(v[e]) * u;
                            }
                        }
                        if constexpr (TY == T_F32)
                            *reinterpret_cast<float4*>(to) = float4{v[0], v[1], v[2], v[3]};
                        else
                            *reinterpret_cast<uint2*>(to) = uint2{i8_half2<TY>(v[0], v[1]), i8_half2<TY>(v[2], v[3])};
                    }
                }
            });
            wave_lds_sync();
#pragma unroll
            for (int p0 = 0; p0 < 32 * PIECES; p0 += 64) {
                const int p = p0 + lane, t = p / PIECES, o = p % PIECES * PER;
                const bool up = GATED && TY < 0 && o >= WR / 2;
                const int n = n0 + (GATED && TY < 0 ? wm * (WR / 2) + o % (WR / 2) : wm * OC + o);
                if (tb + t >= g.T) continue;
                const uint8_t* from = mine + t * PITCH + o * ES;
                uint8_t* to = out + (uint64_t)(tb + t) * pitch + ((uint64_t)n + (up ? g.n_out : 0)) * ES;
                if (n + PER <= g.n_out) {
                    const i8x16 v = *reinterpret_cast<const i8x16*>(from);
                    __builtin_memcpy(to, &v, 16);
                } else {
                    for (int e = 0; e < PER; ++e)
                        if (n + e < g.n_out) {
                            if constexpr (ES == 4)
                                ((uint32_t*)to)[e] = ((const uint32_t*)from)[e];
                            else
                                ((uint16_t*)to)[e] = ((const uint16_t*)from)[e];
                        }
                }
            }
            wave_lds_sync();
            __builtin_amdgcn_sched_barrier(0);  // (the sums of one token tile at a time in vector registers)
        });
    }
}

// The tiles, weight rows x tokens.
enum : int { TILE_256x256 = 0, TILE_128x128 = 1, TILE_128x64 = 2, TILE_64x64 = 3, TILES = 4 };
static const int TILE_M[TILES] = {256, 128, 128, 64}, TILE_N[TILES] = {256, 128, 64, 64};

I8Pick i8_gemm_pick(int rows_w, int k, int T, int gated) {
    (void)gated;
    I8Pick p{TILE_64x64, 1};
    for (int i = 0; i < TILES; ++i) {
        p.tile = i;
        const int64_t tiles = (int64_t)((T + TILE_N[i] - 1) / TILE_N[i]) * ((rows_w + TILE_M[i] - 1) / TILE_M[i]);
        if (tiles >= 200) return p;
    }
    const int64_t tiles = (int64_t)((T + 63) / 64) * ((rows_w + 63) / 64);
    const int stages = (int)(i8_padded(k) / I8_LINE);
    int s = (int)(256 / tiles);
    if (s > stages / 4) s = stages / 4;
    p.splits = s < 1 ? 1 : s;
    return p;
}

bool i8_gemm_reaches(int tile, const I8Args& a) { return (uint64_t)TILE_M[tile] * a.ldw < (1ull << 31); }

template <int WM, int WN, int MT, int NT, int GATED, int TY>
static void launch_as(const I8Args& a, hipStream_t stream) {
    using C = I8Tile<WM, WN, MT, NT>;
    const int bm = GATED ? C::BM / 2 : C::BM;
    const int tw = (a.n_out + bm - 1) / bm, tt = (a.T + C::BN - 1) / C::BN;
    static const hipError_t lds = hipFuncSetAttribute((const void*)k_i8_gemm<WM, WN, MT, NT, GATED, TY>,
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
    (void)lds;  // a launch that the runtime refuses is reported by the caller
    hipLaunchKernelGGL((k_i8_gemm<WM, WN, MT, NT, GATED, TY>), dim3((uint32_t)tw * (uint32_t)tt, 1, a.splits),
                       dim3(64 * C::NW), C::LDS, stream, a, tw, tt);
}
template <int WM, int WN, int MT, int NT, int GATED>
static void launch_gated(const I8Args& a, hipStream_t stream) {
    if (a.splits > 1)
        launch_as<WM, WN, MT, NT, GATED, -1>(a, stream);
    else if (a.ytype == T_F32)
        launch_as<WM, WN, MT, NT, GATED, T_F32>(a, stream);
    else if (a.ytype == T_F16)
        launch_as<WM, WN, MT, NT, GATED, T_F16>(a, stream);
    else
        launch_as<WM, WN, MT, NT, GATED, T_BF16>(a, stream);
}
template <int WM, int WN, int MT, int NT>
static void launch_tile(const I8Args& a, hipStream_t stream) {
    a.gated ? launch_gated<WM, WN, MT, NT, 1>(a, stream) : launch_gated<WM, WN, MT, NT, 0>(a, stream);
}

void launch_i8_gemm(int tile, const I8Args& a, hipStream_t stream) {
    switch (tile) {
    case TILE_256x256: launch_tile<2, 2, 4, 4>(a, stream); break;
    case TILE_128x128: launch_tile<2, 2, 2, 2>(a, stream); break;
    case TILE_128x64: launch_tile<2, 2, 2, 1>(a, stream); break;
    default: launch_tile<1, 2, 2, 1>(a, stream); break;
    }
}

}  // namespace syn
