// The int8 product at many tokens on v_mfma_i32_32x32x32_i8.
//
// A workgroup takes a tile of 32 MT WM weight rows x 32 NT WN tokens; WM x WN x WK wavefronts take 32 MT x 32 NT
// of it each, and a WK-th of K: 64 values of every row a stage and wavefront.  The stages' lines are copied into
// a ring in LDS by global_load_lds, RING - 1 stages ahead.  Piece p (16 bytes) of line r lies at p ^ (r & 7) (p
// ^ (r / 2 & 3) for lines of 64 bytes), so that eight neighbouring lines' same pieces are on eight different
// bank groups.
// Each half stage's operands are read into registers during the half stage before, the first half of the next
// stage's behind the stage's one barrier, and all of it (products, reads, copies) is written in the order in
// which it is to be issued and held there: a large tile leaves two wavefronts a SIMD, of which each has to cover
// its own reads.  Left to itself the compiler reads each operand right before its product (14336 x 4096 at 2048
// tokens 133 us against 130).
// What bounds the large ones is the chip's power: 8192 x 8192 x 8192 of random codes runs at 2240 TOP/s, of zeros
// at 3130; priorities of wavefronts, other orders and deeper rings are within 2 % of it.
// The weight rows are the instruction's A rows, the tokens its columns: a lane holds four neighbouring outputs
// of a token at a time, which go through LDS to whole 16-byte pieces of y's rows.
// WK > 1: for few tokens, where the weights' bytes bound it: more of a small tile's K is in flight, in longer
// pieces of each row.  The wavefronts' sums, whole numbers, meet in LDS and each takes some of the tiles.
// GATED: a wavefront's rows are half gate rows, half the same up rows, so that it holds both values.
// Where the tiles are too few to fill the chip, K is split over gridDim.z workgroups too: whole-number partial
// sums to the workspace, added by k_i8_fold.
#include "int8.hpp"
#include "kernels.hpp"

namespace syn {

template <int N, class F, int I = 0>
SYN_DEV void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<N, F, I + 1>(static_cast<F&&>(f));
    }
}

template <int WM_, int WN_, int WK_, int MT_, int NT_, int RING_>
struct I8Tile {
    static constexpr int WM = WM_, WN = WN_, WK = WK_, MT = MT_, NT = NT_, RING = RING_;
    static constexpr int NW = WM * WN * WK, BM = 32 * MT * WM, BN = 32 * NT * WN;
    static constexpr int LINE = 64 * WK, PIECES = LINE / 16;       // a row's bytes a stage
    static constexpr int RPC = 64 / PIECES;                        // rows a copy instruction
    static constexpr int WPW = BM / RPC / NW, XPW = BN / RPC / NW;  // a wavefront's copies a stage
    static constexpr int CPW = WPW + XPW;
    static constexpr int C0 = CPW / 2;                             // of them issued in a stage's first half
    static constexpr int STAGE = (BM + BN) * LINE;
    // WK > 1: the wavefronts' sums; then a wavefront's outputs of 32 tokens on their way out, its rows' scales
    // and biases
    static constexpr int SUMS = WK > 1 ? NW * MT * NT * 4096 : 0;
    static constexpr int OUT = 32 * (32 * (WK > 1 ? 1 : MT) * 4 + 16) + 32 * MT * 8;
    static constexpr int LDS = RING * STAGE > SUMS + NW * OUT ? RING * STAGE : SUMS + NW * OUT;
    static_assert(BM % (RPC * NW) == 0 && BN % (RPC * NW) == 0, "every wavefront copies as many lines");
    static_assert(WK < 4 || NW % 2 == 0, "a wavefront's copies begin at rows of one parity");
    static_assert(RING >= 3 && CPW * (RING - 2) < 64, "vmcnt");
    static_assert(MT * NT >= 2, "reads beside one product, copies beside another");
    static_assert(LDS <= 160 * 1024, "LDS");
};

template <class C, int GATED, int TY>
__global__ __launch_bounds__(64 * C::NW, C::MT* C::NT >= 16 ? 1 : 2) void k_i8_gemm(I8Args g, int tiles_w, int tiles_t) {
    constexpr int WN = C::WN, WK = C::WK, MT = C::MT, NT = C::NT, RING = C::RING, LINE = C::LINE;
    static_assert(!GATED || MT % 2 == 0, "gate rows and up rows");
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % WN, wm = wave / WN % C::WM, wk = wave / (WN * C::WM);
    const int c = lane & 31, h = lane >> 5;
    int tw, tt;
    i8_tile_of((int)blockIdx.x, tiles_w, tiles_t, tw, tt);
    const int t0 = tt * C::BN;
    const int n0 = tw * (GATED ? C::BM / 2 : C::BM);
    const int kp = (int)i8_padded(g.k), stages = kp / LINE;
    const int z = (int)blockIdx.z;
    const int s0 = (int)((int64_t)stages * z / g.splits), s1 = (int)((int64_t)stages * (z + 1) / g.splits);

    // this wavefront's copies: rows RPC (wave + NW i) .. + RPC - 1, lane l row l / PIECES, place l % PIECES of it
    auto swizzle = [](int r) { return WK == 1 ? (r >> 1) & 3 : r & 7; };
    const int crow = lane / C::PIECES;
    const uint32_t piece = 16u * (uint32_t)((lane % C::PIECES) ^ swizzle(C::RPC * (wave & 1) + crow));
    uint32_t wo[C::WPW], xo[C::XPW];
    const int8_t* wb[GATED ? 2 : 1];
    const int8_t* xb = g.xq + (uint64_t)t0 * kp;
    wb[0] = g.w + (uint64_t)n0 * g.ldw;
    if constexpr (GATED) wb[1] = wb[0] + (uint64_t)g.n_out * g.ldw;
    constexpr int WR = 32 * MT;  // a wavefront's rows
    auto up_half = [&](int i) { return GATED && C::RPC * (wave + C::NW * i) % WR >= WR / 2; };  // uniform
#pragma unroll
    for (int i = 0; i < C::WPW; ++i) {
        const int l = C::RPC * (wave + C::NW * i) + crow;
        int n = GATED ? l / WR * (WR / 2) + l % (WR / 2) : l;
        n = n0 + n < g.n_out ? n : g.n_out - 1 - n0;
        wo[i] = (uint32_t)n * (uint32_t)g.ldw + piece;
    }
#pragma unroll
    for (int i = 0; i < C::XPW; ++i) {
        int t = C::RPC * (wave + C::NW * i) + crow;
        t = t0 + t < g.T ? t : g.T - 1 - t0;
        xo[i] = (uint32_t)t * (uint32_t)kp + piece;
    }
    const uint32_t ring = lds_addr(lds);
    const int whole = g.k / LINE;                          // stages that every weight row fills
    const uint32_t lastp = (uint32_t)(g.k - 1) & ~15u;     // a row's last piece
    // What the copies of stage s share: the ring's place for it, and where it lies in a row.  Past a weight
    // row's end its last piece again, against zeros.  Past the part's last stage that one again, into places
    // that are read by nothing that counts: the loop has one form.
    struct Where {
        uint32_t to, adj;
        uint64_t w, x;
    };
    auto where = [&](int s, int place) {
        Where v;
        v.to = ring + (uint32_t)place * C::STAGE;
        s = s < s1 ? s : s1 - 1;
        const uint32_t p = (uint32_t)s * LINE + piece;
        v.adj = s < whole ? 0u : (p < lastp ? p : lastp) - piece;
        v.w = s < whole ? (uint64_t)s * LINE : 0u;
        v.x = (uint64_t)s * LINE;
        return v;
    };
    // copy i of a stage: the weight rows' first, then the tokens'
    auto copy = [&](const Where& v, int i) {
        if (i < C::WPW) {
            const int j = i < C::WPW ? i : 0;
            lds_dma16(wo[j] + v.adj, wb[up_half(j)] + v.w, v.to + 1024u * (uint32_t)(wave + C::NW * j));
        } else {
            const int j = i - C::WPW;
            lds_dma16(xo[j], xb + v.x, v.to + C::BM * LINE + 1024u * (uint32_t)(wave + C::NW * j));
        }
    };

    i32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = i32x16{};

    i8x16 a[2][MT], b[2][NT];
    const int place = 16 * ((4 * wk + h) ^ swizzle(c));  // of piece 4 wk + h; piece 4 wk + 2 + h lies at place ^ 32
    const uint8_t* al = lds + (wm * WR + c) * LINE;
    const uint8_t* bl = lds + C::BM * LINE + (wn * 32 * NT + c) * LINE;
    // operand r of half kk of the stage at `at` of the ring into buffer kk
    auto read = [&](int at, int kk, int r) {
        const int off = at * C::STAGE + (place ^ (32 * kk));
        if (r < MT)
            a[kk][r < MT ? r : 0] = *reinterpret_cast<const i8x16*>(al + off + (r < MT ? r : 0) * 32 * LINE);
        else
            b[kk][r - MT] = *reinterpret_cast<const i8x16*>(bl + off + (r - MT) * 32 * LINE);
    };
    // the products of half kk, the reads of the other buffer's half and half of a stage's copies among them
    auto half = [&](auto kkc, int rs, const Where& v) {
        constexpr int kk = decltype(kkc)::value;
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

    static_for<RING - 1>([&](auto sc) {
        const Where v = where(s0 + decltype(sc)::value, decltype(sc)::value);
        static_for<C::CPW>([&](auto i) { copy(v, decltype(i)::value); });
    });
    wait_vm<(RING - 2) * C::CPW>();
    lds_barrier();
    static_for<MT + NT>([&](auto r) { read(0, 0, decltype(r)::value); });
    int at = 0, to = RING - 1;  // the ring's places of stage s, and of what is copied during it
    for (int s = s0; s < s1; ++s) {
        const Where v = where(s + RING - 1, to);
        half(std::integral_constant<int, 0>{}, at, v);
        wait_vm<(RING - 3) * C::CPW + C::C0>();  // stage s + 1 is there
        lds_barrier();
        to = at;
        at = at + 1 == RING ? 0 : at + 1;
        half(std::integral_constant<int, 1>{}, at, v);
    }
    wait_vm<0>();
    lds_barrier();  // the ring is free

    // lane: token c of each tile of 32, rows 8 e4 + 4 h + 0..3
    uint8_t* mine = lds + C::SUMS + wave * C::OUT;
    float* sw = reinterpret_cast<float*>(mine + C::OUT - 8 * WR);  // [WR], then the biases
    if constexpr (TY >= 0) {
        for (int r = lane; r < WR; r += 64) {
            int n = n0 + (GATED ? wm * (WR / 2) + r % (WR / 2) : wm * WR + r);
            n = (n < g.n_out ? n : g.n_out - 1) + (GATED && r >= WR / 2 ? g.n_out : 0);
            sw[r] = g.ws[n];
            sw[WR + r] = g.bias ? g.bias[n] : 0.0f;
        }
        wave_lds_sync();
    }
    // TY: an output type, or -1: the sums of a part of K
    constexpr int ES = TY == T_F32 || TY < 0 ? 4 : 2;
    constexpr int HALVES = GATED && TY >= 0 ? 2 : 1;  // of a wavefront's rows that make one output together
    const uint64_t rows_w = (uint64_t)g.n_out * (GATED ? 2 : 1);
    uint8_t* out = TY < 0 ? (uint8_t*)(g.partial + (uint64_t)z * g.T * rows_w) : (uint8_t*)g.y;
    const uint64_t pitch = (TY < 0 ? rows_w : g.ldy) * ES;
    // the outputs of token tile j, row tiles i0 .. i0 + IC - 1
    auto emit = [&](auto jc, auto i0c, auto icc) {
        constexpr int j = decltype(jc)::value, i0 = decltype(i0c)::value, IC = decltype(icc)::value;
        constexpr int OC = 32 * IC, PITCH = OC * ES + 16, PIECES = OC * ES / 16, PER = 16 / ES;
        const int tb = t0 + (wn * NT + j) * 32;
        const float sx = g.xs[tb + c];
        static_for<IC>([&](auto ic) {
            constexpr int i = i0 + decltype(ic)::value;
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int o = i * 32 + 8 * e4 + 4 * h;  // of the wavefront's rows
                uint8_t* to = mine + c * PITCH + (o - 32 * i0) * ES;
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
            const int p = p0 + lane, t = p / PIECES, o = 32 * i0 + p % PIECES * PER;  // o: of the wavefront's rows
            const bool up = GATED && o >= WR / 2;
            const int n = n0 + (GATED ? wm * (WR / 2) + o % (WR / 2) : wm * WR + o);
            if (tb + t >= g.T) continue;
            const uint8_t* from = mine + t * PITCH + (o - 32 * i0) * ES;
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
    };
    if constexpr (WK == 1) {
        static_for<NT>([&](auto jc) {
            emit(jc, std::integral_constant<int, 0>{}, std::integral_constant<int, MT / HALVES>{});
        });
    } else {
        // output tile u goes to the wavefront of part u % WK: the others' sums of it through LDS
        constexpr int RT = MT / HALVES;  // row tiles of outputs
        auto area = [&](int part, int i, int j) {
            return reinterpret_cast<i8x16*>(lds) + ((((part * C::WM + wm) * WN + wn) * MT + i) * NT + j) * 256 + lane;
        };
        static_for<MT * NT>([&](auto uc) {
            constexpr int u = decltype(uc)::value, i = u / NT, j = u % NT;
            if ((i % RT * NT + j) % WK == wk) return;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                area(wk, i, j)[64 * e] = i8x16{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
        });
        lds_barrier();
        static_for<RT * NT>([&](auto uc) {
            constexpr int u = decltype(uc)::value, j = u % NT;
            if (u % WK != wk) return;  // uniform
            static_for<HALVES>([&](auto hc) {
                constexpr int i = u / NT + decltype(hc)::value * RT;
#pragma unroll
                for (int q = 1; q < WK; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const i8x16 v = area((wk + q) % WK, i, j)[64 * e];
#pragma unroll
                        for (int m = 0; m < 4; ++m) acc[i][j][4 * e + m] += v[m];
                    }
            });
            emit(std::integral_constant<int, j>{}, std::integral_constant<int, u / NT>{}, std::integral_constant<int, 1>{});
        });
    }
}

// The tiles: wavefronts over weight rows, tokens and K, each one's 32-row and 32-token tiles, the ring's stages;
// then what a workgroup that has a CU to itself takes beside K and a 1024 values of K, in tenths of a
// microsecond (product alone, 256 workgroups: 4096 x 4096 and 4096 x 14336 matrices at 128 to 2048 tokens).
// Every tile's ring leaves room for one workgroup a CU.
// Of 41 calls over matrices of 1024 to 32064 rows at 17 to 3900 tokens 36 run on the fastest tile, the others within
// 8 % of it (profiles/int8_products_and_token_logprobs.md).
#define SYN_I8_TILES(X)              \
    X(0, 4, 2, 1, 2, 4, 4, 50, 147)  \
    X(1, 4, 2, 1, 2, 2, 4, 27, 100)  \
    X(2, 2, 4, 1, 2, 2, 4, 30, 87)   \
    X(3, 2, 4, 1, 2, 1, 6, 5, 60)    \
    X(4, 2, 1, 2, 2, 4, 3, 56, 48)   \
    X(5, 1, 2, 2, 2, 2, 4, 2, 32)    \
    X(6, 1, 1, 4, 2, 2, 4, 4, 20)    \
    X(7, 1, 1, 4, 2, 1, 4, 1, 15)
struct TileOf {
    int m, n;          // weight rows, tokens
    float base, per_k;  // microseconds a workgroup, and a value of K
};
#define SYN_I8_TILE(id, wm, wn, wk, mt, nt, ring, base, k) {32 * wm * mt, 32 * wn * nt, 0.1f * base, 0.1f * k / 1024},
static const TileOf TILES[] = {SYN_I8_TILES(SYN_I8_TILE)};
#undef SYN_I8_TILE

// The tile and the parts of K that are estimated to take least: rounds of 256 workgroups, the last one's a
// little faster the fewer there are in it, beside what the weights take from HBM (4.9 TB/s at most, 45 GB/s a
// workgroup, and part of a reading more for every further tile of tokens): the longer of the two and a quarter
// of the other; K in parts costs the fold's launch and its partial sums' writing and reading.  Large tiles read less from L2 for an output,
// small ones fill the chip: 4096 x 4096 at 512 tokens takes 16 us in 256 tiles of 64 x 128 and 50 in 32 of 256
// x 256, 14336 x 4096 at 2048 tokens 133 in 448 of 256 x 256 and 167 in 1792 of 128 x 128; 4096 x 14336 at 64
// tokens 19 in 64 tiles of 64 x 64 of a quarter of K each and 27 in 128 of 64 x 32 of a half.
I8Pick i8_gemm_pick(int rows_w, int k, int T) {
    constexpr float LAUNCH = 3.0f, FOLD = 3.5f;                     // us
    constexpr float HBM = 4.9e6f, EACH = 4.5e4f, SUMS = 4.0e6f;     // bytes a us
    const int kp = (int)i8_padded(k);
    I8Pick best{0, 1};
    if (rows_w == 0) return best;  // nothing to estimate (0 / 0)
    float least = 0.0f;
    for (int i = 0; i < (int)(sizeof TILES / sizeof TILES[0]); ++i) {
        const TileOf& t = TILES[i];
        const int64_t tw = (rows_w + t.m - 1) / t.m, tt = (T + t.n - 1) / t.n;
        const float bytes = (float)rows_w * (float)k * (tt < 4 ? 0.6f + 0.4f * (float)tt : 2.0f);
        for (int s = 1; s <= 8; s = s < 4 ? s + 1 : s + 2) {
            const int64_t wgs = tw * tt * s, rounds = (wgs + 255) / 256;
            if (s > 1 && (kp < 1024 * s || wgs > 256)) break;  // (a part has four stages and more)
            const float last = (float)(wgs - 256 * (rounds - 1)) / 256.0f, turns = (float)rounds - 0.25f + 0.25f * last;
            const float work = (float)rounds * t.base + turns * t.per_k * (float)kp / (float)s;
            const float rate = EACH * (float)wgs < HBM ? EACH * (float)wgs : HBM;
            const float read = bytes / rate;
            float us = LAUNCH + (work > read ? work + 0.25f * read : read + 0.25f * work);  // (they overlap in part)
            if (s > 1) us += FOLD + 8.0f * (float)s * (float)T * (float)rows_w / SUMS;
            if (least == 0.0f || us < least) {
                least = us;
                best = I8Pick{i, s};
            }
        }
    }
    return best;
}

bool i8_gemm_reaches(int tile, const I8Args& a) { return (uint64_t)TILES[tile].m * a.ldw < (1ull << 31); }

template <class C, int GATED, int TY>
static void launch_as(const I8Args& a, hipStream_t stream) {
    const int bm = GATED ? C::BM / 2 : C::BM;
    const int tw = (a.n_out + bm - 1) / bm, tt = (a.T + C::BN - 1) / C::BN;
    static std::atomic<uint64_t> said{0};
    i8_allow_lds((const void*)k_i8_gemm<C, GATED, TY>, C::LDS, said);
    hipLaunchKernelGGL((k_i8_gemm<C, GATED, TY>), dim3((uint32_t)tw * (uint32_t)tt, 1, a.splits), dim3(64 * C::NW), C::LDS,
                       stream, a, tw, tt);
}
template <class C, int GATED>
static void launch_gated(const I8Args& a, hipStream_t stream) {
    if (a.splits > 1)
        launch_as<C, GATED, -1>(a, stream);
    else if (a.ytype == T_F32)
        launch_as<C, GATED, T_F32>(a, stream);
    else if (a.ytype == T_F16)
        launch_as<C, GATED, T_F16>(a, stream);
    else
        launch_as<C, GATED, T_BF16>(a, stream);
}

void launch_i8_gemm(int tile, const I8Args& a, hipStream_t stream) {
#define SYN_I8_CASE(id, wm, wn, wk, mt, nt, ring, base, k)                     \
    case id:                                                                   \
        a.gated ? launch_gated<I8Tile<wm, wn, wk, mt, nt, ring>, 1>(a, stream) \
                : launch_gated<I8Tile<wm, wn, wk, mt, nt, ring>, 0>(a, stream); \
        break;
    switch (tile) { SYN_I8_TILES(SYN_I8_CASE) }
#undef SYN_I8_CASE
}

}  // namespace syn
