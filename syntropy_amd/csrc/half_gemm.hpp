// The half-precision product at many tokens on v_mfma_f32_32x32x16.
//
// A workgroup takes a tile of 32 MT WM weight rows x 32 NT WN tokens; WM x WN x WK wavefronts take 32 MT x 32 NT
// of it each, and a WK-th of K: 32 values of every row a stage and wavefront.  The stages' lines are copied into
// a ring in LDS by global_load_lds, RING - 1 stages ahead (RING 0: whole lines of 128 bytes, two stages and a half
// ahead, below).  Piece p (16 bytes) of line r lies at p ^ (r & 7) (p
// ^ (r / 2 & 3) for lines of 64 bytes), so that eight neighbouring lines' same pieces are on eight different
// bank groups.
// Each half stage's operands are read into registers during the half stage before, the first half of the next
// stage's behind the stage's one barrier, and all of it (products, reads, copies) is written in the order in
// which it is to be issued and held there: a large tile leaves one or two wavefronts a SIMD, of which each has to cover
// its own reads.  Bound by the matrix cores at many tokens: 8192^3 takes 790 us (1390 TFLOP/s; the library's product
// 767), 14336 x 4096 at 2048 tokens 200 (1200 TFLOP/s; 203), where 448 tiles are two rounds over 256 CUs for 1.75.
// The weight rows are the instruction's A rows, the tokens its columns: a lane holds four neighbouring outputs
// of a token at a time, which go, with the bias, through LDS to whole pieces of y's rows, where the activation is
// applied and gate and residual are read as such pieces too.
// WK > 1: for few tokens, where the weights' bytes bound it: more of a small tile's K is in flight, in longer
// pieces of each row.  The wavefronts' sums meet in LDS, in a fixed order, and each takes some of the tiles.
// Where the tiles are too few to fill the chip, K is split over gridDim.z workgroups too: partial sums to the
// workspace, added in order by k_half_fold.
#pragma once

#include "half.hpp"
#include "kernels.hpp"

namespace syn {

template <int WM_, int WN_, int WK_, int MT_, int NT_, int RING_>
struct HalfTile {
    static constexpr int WM = WM_, WN = WN_, WK = WK_, MT = MT_, NT = NT_, RING = RING_;
    static constexpr bool WIDE = RING == 0;
    static constexpr int NW = WM * WN * WK, BM = 32 * MT * WM, BN = 32 * NT * WN;
    static constexpr int LINE = WIDE ? 128 : 64 * WK, PIECES = LINE / 16;  // a row's bytes a stage
    static constexpr int RPC = 64 / PIECES;                        // rows a copy instruction
    static constexpr int WPW = BM / RPC / NW, XPW = BN / RPC / NW;  // a wavefront's copies a stage
    static constexpr int CPW = WPW + XPW;
    static constexpr int C0 = CPW / 2;                             // of them issued in a stage's first half
    static constexpr int STAGE = (BM + BN) * LINE;
    static constexpr int UNIT = BM * LINE;                         // WIDE: of five, the weight rows or the tokens of a stage
    static constexpr int COPIES = WIDE ? 5 * UNIT : RING * STAGE;
    // WK > 1: the wavefronts' sums; then a wavefront's outputs of 32 tokens on their way out, its rows' biases
    static constexpr int SUMS = WK > 1 ? NW * MT * NT * 4096 : 0;
    static constexpr int OUT = 32 * (32 * (WK > 1 ? 1 : MT) * 4 + 16) + 32 * MT * 4;
    static constexpr int LDS = COPIES > SUMS + NW * OUT ? COPIES : SUMS + NW * OUT;
    static_assert(BM % (RPC * NW) == 0 && BN % (RPC * NW) == 0, "every wavefront copies as many lines");
    static_assert(PIECES < 8 || NW % 2 == 0 || WIDE, "a wavefront's copies begin at rows of one parity");
    static_assert(WIDE || (RING >= 3 && CPW * (RING - 2) < 64), "vmcnt");
    static_assert(!WIDE || (WK == 1 && BM == BN && XPW == WPW && WPW <= MT * NT && MT + NT <= MT * NT), "copies and reads beside products");
    static_assert(LDS <= 160 * 1024, "LDS");
    static_assert(2 * HALF_PAIR % LINE == 0, "a row is whole stages");
};

enum HalfOut { OUT_PART, OUT_F32, OUT_16 };  // the sums of a part of K; F32; F16 or BF16

template <class C, int WTY, int OT>
__global__ __launch_bounds__(64 * C::NW, 2) void k_half_gemm(HalfArgs g, int tiles_w, int tiles_t) {
    constexpr int WN = C::WN, WK = C::WK, MT = C::MT, NT = C::NT, RING = C::RING, LINE = C::LINE;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave % WN, wm = wave / WN % C::WM, wk = wave / (WN * C::WM);
    const int c = lane & 31, h = lane >> 5;
    int tw, tt;
    i8_tile_of((int)blockIdx.x, tiles_w, tiles_t, tw, tt);
    const int t0 = tt * C::BN, n0 = tw * C::BM;
    const int stages = (int)(2 * half_padded(g.k) / LINE);
    const int z = (int)blockIdx.z;
    const int s0 = (int)((int64_t)stages * z / g.splits), s1 = (int)((int64_t)stages * (z + 1) / g.splits);

    // this wavefront's copies: rows RPC (wave + NW i) .. + RPC - 1, lane l row l / PIECES, place l % PIECES of it
    auto swizzle = [](int r) { return C::PIECES == 4 ? (r >> 1) & 3 : r & 7; };
    const int crow = lane / C::PIECES;
    const uint32_t piece = 16u * (uint32_t)((lane % C::PIECES) ^ swizzle(C::RPC * (wave & 1) + crow));
    uint32_t wo[C::WPW], xo[C::XPW];
    const uint8_t* wb = (const uint8_t*)(g.w + (uint64_t)n0 * g.ldw);
    const uint8_t* xb = (const uint8_t*)(g.x + (uint64_t)t0 * g.ldx);
#pragma unroll
    for (int i = 0; i < C::WPW; ++i) {
        int n = C::RPC * (wave + C::NW * i) + crow;
        n = n0 + n < g.n_out ? n : g.n_out - 1 - n0;
        wo[i] = (uint32_t)n * (uint32_t)(2 * g.ldw) + piece;
    }
#pragma unroll
    for (int i = 0; i < C::XPW; ++i) {
        int t = C::RPC * (wave + C::NW * i) + crow;
        t = t0 + t < g.T ? t : g.T - 1 - t0;
        xo[i] = (uint32_t)t * (uint32_t)(2 * g.ldx) + piece;
    }
    const uint32_t ring = lds_addr(lds);
    // What the copies of stage s share: the ring's place for it, and where it lies in a row.  Past the part's last
    // stage that one again, into places that are read by nothing that counts: the loop has one form.
    struct Where {
        uint32_t to;
        uint64_t at;
    };
    auto where = [&](int s, int place) {
        return Where{ring + (uint32_t)place * C::STAGE, (uint64_t)(s < s1 ? s : s1 - 1) * LINE};
    };
    // copy i of a stage: the weight rows' first, then the tokens'
    auto copy = [&](const Where& v, int i) {
        if (i < C::WPW) {
            const int j = i < C::WPW ? i : 0;
            lds_dma16(wo[j], wb + v.at, v.to + 1024u * (uint32_t)(wave + C::NW * j));
        } else {
            const int j = i - C::WPW;
            lds_dma16(xo[j], xb + v.at, v.to + C::BM * LINE + 1024u * (uint32_t)(wave + C::NW * j));
        }
    };

    f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x16{};

    i8x16 a[2][MT], b[2][NT];
    const int place = 16 * ((4 * wk + h) ^ swizzle(c));  // of piece 4 wk + h; piece 4 wk + 2 + h lies at place ^ 32
    constexpr int WR = 32 * MT;                          // a wavefront's rows
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
            acc[i][j] = half_mfma32<WTY>(a[kk][i], b[kk][j], acc[i][j]);
            // reads in the first half of the products (one or more a product), copies in the second
            constexpr int H = M > 1 ? M / 2 : 1;
            constexpr int r0 = m < H ? m * R / H : R, r1 = m < H ? (m + 1) * R / H : R;
            if constexpr (r1 > r0) static_for<r1 - r0>([&](auto rc) { read(rs, 1 - kk, r0 + decltype(rc)::value); });
            constexpr int L = M > 1 ? M - H : 1, l = M > 1 ? m - H : 0;
            constexpr int c0 = l >= 0 ? l * CP / L : 0, c1 = l >= 0 ? (l + 1) * CP / L : 0;
            if constexpr (c1 > c0) static_for<c1 - c0>([&](auto cc) { copy(v, first + c0 + decltype(cc)::value); });
            __builtin_amdgcn_sched_barrier(0);
        });
    };

    // What the epilogue reads of gate and residual is fetched a group of pieces ahead, the first group before all else.  Within
    // a unit a group is under way beside the one before.  A unit's first group is not: the wait for LDS at the end of the
    // unit before is one for all memory, that unit's stores too.  (F32 operands of an output of 16 bits, twice as
    // long, are not fetched ahead.)
    constexpr int IC = WK > 1 ? 1 : MT;                           // row tiles of an emission
    constexpr int OC = 32 * IC, PITCH = OC * 4 + 16;
    constexpr int PER = OT == OUT_16 ? 8 : 4, ROW = OC / PER;     // values of 16 bytes, pieces a token
    constexpr int TURNS = 32 * ROW / 64, GROUP = TURNS < 4 ? TURNS : 4, GROUPS = TURNS / GROUP;
    static_assert(64 % ROW == 0, "the same outputs each turn");
    HalfRaw<PER> gates[GROUP] = {}, sums[GROUP] = {};
    const bool gates_ahead = g.gate && (OT == OUT_F32 || g.gtype != T_F32), res_ahead = g.res && (OT == OUT_F32 || g.rtype != T_F32);
    const int lo = lane % ROW * PER;                              // of the emission's outputs
    auto fetch = [&](int i0, int j, int gi) {
        if constexpr (OT != OUT_PART) {
            if (!gates_ahead && !res_ahead) return;  // uniform
            const int tb = t0 + (wn * NT + j) * 32, nb = n0 + wm * 32 * MT + 32 * i0;
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                const int t = tb + (64 * (GROUP * gi + q) + lane) / ROW;
                if (t >= g.T || nb + lo + PER > g.n_out) continue;
                if (gates_ahead) half_fetch<PER>(g.gate, g.gtype, (uint64_t)t * g.ldg + nb + lo, gates[q]);
                if (res_ahead) half_fetch<PER>(g.res, g.rtype, (uint64_t)t * g.ldr + nb + lo, sums[q]);
            }
        }
    };
    if constexpr (WK == 1) {
        fetch(0, 0, 0);
    } else {
        static_assert(MT * NT % WK == 0 || MT * NT < WK, "as many tiles a part");
        if (wk < MT * NT) fetch(wk / NT, wk % NT, 0);
    }

    if constexpr (C::WIDE) {
        // Whole 128-byte lines, 64 values of every row a stage, its weight rows and its tokens a unit each, unit u in place
        // u % 5.  Behind the stage's one barrier, before its last quarter, both of its units are free: the tokens of
        // the stage after next are copied to the first beside that quarter, the weight rows of the third to the
        // second beside the next stage's first two.
        auto place5 = [](int u) { return u >= 5 ? u - 5 : u; };
        // where the stage's lines begin (a scalar, said to be one: the copies' base is); past the part's last stage that
        // one's again
        auto from = [&](const uint8_t* base, int s) {
            const uint64_t p = (uint64_t)(uintptr_t)base + (uint64_t)(s < s1 ? s : s1 - 1) * LINE;
            const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p);
            const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32));
            return (const uint8_t*)(uintptr_t)((uint64_t)hi << 32 | lo);
        };
        // copy i of a unit's into its place
        auto copy5 = [&](const uint8_t* base, const uint32_t (&offsets)[C::WPW], int slot, int i) {
            lds_dma16(offsets[i], base, ring + (uint32_t)slot * C::UNIT + 1024u * (uint32_t)(wave + C::NW * i));
        };
        const uint8_t* aw = lds + (wm * WR + c) * LINE;
        const uint8_t* bx = lds + (wn * 32 * NT + c) * LINE;
        auto operand = [&](int slot, int q, int r) {
            const int off = 16 * ((2 * q + h) ^ (c & 7));
            if (r < MT)
                a[q & 1][r < MT ? r : 0] = *reinterpret_cast<const i8x16*>(aw + slot * C::UNIT + off + (r < MT ? r : 0) * 32 * LINE);
            else
                b[q & 1][r - MT] = *reinterpret_cast<const i8x16*>(bx + place5(slot + 1) * C::UNIT + off + (r - MT) * 32 * LINE);
        };
        // the products of quarter q, the reads of the next one's operands (of the stage at `slot`) and copies among them
        auto quarter = [&](auto qc, int slot, auto&& copies) {
            constexpr int q = decltype(qc)::value, M = MT * NT, R = MT + NT;
            static_for<M>([&](auto mc) {
                constexpr int m = decltype(mc)::value, i = m / NT, j = m % NT;
                acc[i][j] = half_mfma32<WTY>(a[q & 1][i], b[q & 1][j], acc[i][j]);
                if constexpr (m < R) operand(slot, (q + 1) & 3, m);
                copies(m);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        static_for<C::WPW>([&](auto i) { copy5(from(wb, s0), wo, 0, decltype(i)::value); });
        static_for<C::WPW>([&](auto i) { copy5(from(xb, s0), xo, 1, decltype(i)::value); });
        static_for<C::WPW>([&](auto i) { copy5(from(wb, s0 + 1), wo, 2, decltype(i)::value); });
        static_for<C::WPW>([&](auto i) { copy5(from(xb, s0 + 1), xo, 3, decltype(i)::value); });
        wait_vm<2 * C::WPW>();
        lds_barrier();
        static_for<MT + NT>([&](auto r) { operand(0, 0, decltype(r)::value); });
        int slot = 0;
        for (int s = s0; s < s1; ++s) {
            const int spare = place5(slot + 4), next = place5(slot + 2);
            const uint8_t *w2 = from(wb, s + 2), *x2 = from(xb, s + 2);
            quarter(std::integral_constant<int, 0>{}, slot, [&](int m) {
                if (m >= MT * NT - C::WPW) copy5(w2, wo, spare, m - (MT * NT - C::WPW));
            });
            quarter(std::integral_constant<int, 1>{}, slot, [](int) {});
            quarter(std::integral_constant<int, 2>{}, slot, [](int) {});
            wait_vm<C::WPW>();  // stage s + 1 is there
            lds_barrier();
            quarter(std::integral_constant<int, 3>{}, next, [&](int m) {
                if (m < C::WPW) copy5(x2, xo, slot, m);
            });
            slot = next;
        }
    } else {
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
    }
    wait_vm<0>();
    lds_barrier();  // the ring is free

    // lane: token c of each tile of 32, rows 8 e4 + 4 h + 0..3
    uint8_t* mine = lds + C::SUMS + wave * C::OUT;
    float* bias = reinterpret_cast<float*>(mine + C::OUT - 4 * WR);  // [WR]
    if constexpr (OT != OUT_PART) {
        if (g.bias) {
            for (int r = lane; r < WR; r += 64) {
                const int n = n0 + wm * WR + r;
                bias[r] = g.bias[n < g.n_out ? n : g.n_out - 1];
            }
            wave_lds_sync();
        }
    }
    // WK > 1: output tile q goes to the wavefront of part q % WK: the others' sums of it through LDS
    auto area = [&](int part, int i, int j) {
        return reinterpret_cast<f32x4*>(lds) + ((((part * C::WM + wm) * WN + wn) * MT + i) * NT + j) * 256 + lane;
    };
    if constexpr (WK > 1) {
        static_for<MT * NT>([&](auto qc) {
            constexpr int q = decltype(qc)::value, i = q / NT, j = q % NT;
            if (q % WK == wk) return;  // uniform
#pragma unroll
            for (int e = 0; e < 4; ++e)
                area(wk, i, j)[64 * e] = f32x4{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
        });
        lds_barrier();
    }
    // The outputs of row tiles i0 .. i0 + IC - 1 of token tile j on their way out, the biases added.  WK > 1: the parts'
    // sums are added in their order, from this wavefront's own on.
    auto stage = [&](auto i0c, auto jc) {
        constexpr int i0 = decltype(i0c)::value, j = decltype(jc)::value;
        static_for<IC>([&](auto ic) {
            constexpr int i = i0 + decltype(ic)::value;
            f32x16 sum = acc[i][j];
            if constexpr (WK > 1) {
#pragma unroll
                for (int q = 1; q < WK; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const f32x4 v = area((wk + q) % WK, i, j)[64 * e];
#pragma unroll
                        for (int m = 0; m < 4; ++m) sum[4 * e + m] += v[m];
                    }
            }
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int o = i * 32 + 8 * e4 + 4 * h;  // of the wavefront's rows
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = sum[4 * e4 + e];
                if constexpr (OT != OUT_PART) {
                    if (g.bias) {
                        const float4 bv = *reinterpret_cast<const float4*>(bias + o);
                        v[0] = v[0] + bv.x, v[1] = v[1] + bv.y, v[2] = v[2] + bv.z, v[3] = v[3] + bv.w;
                    }
                }
                *reinterpret_cast<float4*>(mine + c * PITCH + (o - 32 * i0) * 4) = float4{v[0], v[1], v[2], v[3]};
            }
        });
    };
    // A unit is what is on its way out at a time.  Only the registers it comes from are a unit's own code, what follows is in it
    // once: a workgroup runs through it once or twice, and with a copy a unit and type the epilogue was 30 to 60 KB (with
    // that, and the residual not fetched ahead beside a gate, 14336 x 4096 at 2048 rows 251 us in place of 234).
    constexpr int UNITS = WK > 1 ? (MT * NT + WK - 1) / WK : NT;
    auto tile_of = [&](int u) { return WK > 1 ? u * WK + wk : u; };
#pragma unroll 1
    for (int u = 0; u < UNITS; ++u) {
        if (WK > 1 && tile_of(u) >= MT * NT) break;  // uniform
        static_for<WK == 1 ? NT : MT * NT>([&](auto qc) {
            constexpr int q = decltype(qc)::value;
            if (q == tile_of(u)) stage(std::integral_constant<int, WK == 1 ? 0 : q / NT>{}, std::integral_constant<int, q % NT>{});
        });
        auto rows_of = [&](int u) { return WK > 1 ? tile_of(u) / NT : 0; };
        auto tokens_of = [&](int u) { return tile_of(u) % NT; };
        const int un = u + 1 < UNITS && (WK == 1 || tile_of(u + 1) < MT * NT) ? u + 1 : u;
        const int i0 = rows_of(u), j = tokens_of(u), tb = t0 + (wn * NT + j) * 32, nb = n0 + wm * WR + 32 * i0;
        wave_lds_sync();
        if constexpr (OT != OUT_PART) {
            // in place, eight values at a time
            half_act_of(g.act, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
#pragma unroll 1
                for (int p = lane; p < 32 * OC / 4; p += 128) {
                    float4* a0 = reinterpret_cast<float4*>(mine + p / (OC / 4) * PITCH) + p % (OC / 4);
                    float4* a1 = a0 + 64 / (OC / 4) * (PITCH / 16);
                    float4 v = *a0, w = *a1;
                    v.x = half_act<ACT>(v.x), v.y = half_act<ACT>(v.y), v.z = half_act<ACT>(v.z), v.w = half_act<ACT>(v.w);
                    w.x = half_act<ACT>(w.x), w.y = half_act<ACT>(w.y), w.z = half_act<ACT>(w.z), w.w = half_act<ACT>(w.w);
                    *a0 = v, *a1 = w;
                }
                wave_lds_sync();
            });
        }
        const float* staged = reinterpret_cast<const float*>(mine);
        // Piece p of the unit: token p / ROW, outputs p % ROW * PER ..  (y may be gate or residual: what a lane writes
        // it has read, and no other lane reads.)
        const int n = nb + lo;
        const bool whole = n + PER <= g.n_out;
#pragma unroll 1
        for (int gi = 0; gi < GROUPS; ++gi) {
            auto token = [&](int q) { return (64 * (GROUP * gi + q) + lane) / ROW; };
            uint32_t out[GROUP][4];
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                const int t = token(q);
                float v[PER];
#pragma unroll
                for (int e = 0; e < PER; e += 4) {
                    const float4 f = *reinterpret_cast<const float4*>(staged + t * (PITCH / 4) + lo + e);
                    v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
                }
                if constexpr (OT != OUT_PART) {
                    float o[PER] = {};
                    if (g.gate) {
                        if (gates_ahead)
                            half_unpack<PER>(g.gtype, gates[q], o);
                        else if (tb + t < g.T && whole)
                            half_load<PER>(g.gate, g.gtype, (uint64_t)(tb + t) * g.ldg + n, PER, o);
#pragma unroll
                        for (int e = 0; e < PER; ++e) v[e] = v[e] * o[e];
                    }
                    if (g.res) {
                        if (res_ahead)
                            half_unpack<PER>(g.rtype, sums[q], o);
                        else if (tb + t < g.T && whole)
                            half_load<PER>(g.res, g.rtype, (uint64_t)(tb + t) * g.ldr + n, PER, o);
#pragma unroll
                        for (int e = 0; e < PER; ++e) v[e] = v[e] + o[e];
                    }
                }
                if constexpr (OT != OUT_16) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[q][e] = f2u(v[e]);
                } else if (g.ytype == T_F16) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[q][e] = i8_half2<T_F16>(v[2 * e], v[2 * e + 1]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) out[q][e] = i8_half2<T_BF16>(v[2 * e], v[2 * e + 1]);
                }
            }
            const bool on = gi + 1 < GROUPS;
            fetch(on ? i0 : rows_of(un), on ? j : tokens_of(un), on ? gi + 1 : 0);
#pragma unroll
            for (int q = 0; q < GROUP; ++q) {
                const int t = token(q);
                if (tb + t >= g.T || !whole) continue;
                if constexpr (OT == OUT_PART)
                    __builtin_memcpy(g.partial + ((uint64_t)z * g.T + tb + t) * (uint64_t)g.n_out + n, out[q], 16);
                else if constexpr (OT == OUT_F32)
                    __builtin_memcpy((float*)g.y + (uint64_t)(tb + t) * g.ldy + n, out[q], 16);
                else
                    __builtin_memcpy((uint16_t*)g.y + (uint64_t)(tb + t) * g.ldy + n, out[q], 16);
            }
        }
        // The outputs behind the last whole piece, value by value, their operands' loads before the first is waited for (all of
        // a ragged tile's outputs in turn took 21 of 39 us of 12976 x 1024 at 256 rows with a residual).
        const int left = g.n_out - nb, e0 = left / PER * PER, ragged = left - e0;
        if (left < OC && ragged > 0) {  // uniform
            constexpr int MOST = (32 * (PER - 1) + 63) / 64;
            float gate[MOST], res[MOST];
            auto place = [&](int m, int& t, int& n) {
                const int p = 64 * m + lane;
                t = p / ragged, n = e0 + p % ragged;
                return t < 32 && tb + t < g.T;
            };
            if constexpr (OT != OUT_PART) {
#pragma unroll
                for (int m = 0; m < MOST; ++m) {
                    int t, n;
                    if (!place(m, t, n)) continue;
                    if (g.gate) gate[m] = half_at(g.gate, g.gtype, (uint64_t)(tb + t) * g.ldg + nb + n);
                    if (g.res) res[m] = half_at(g.res, g.rtype, (uint64_t)(tb + t) * g.ldr + nb + n);
                }
            }
#pragma unroll
            for (int m = 0; m < MOST; ++m) {
                int t, n;
                if (!place(m, t, n)) continue;
                float v = staged[t * (PITCH / 4) + n];
                if constexpr (OT == OUT_PART) {
                    g.partial[((uint64_t)z * g.T + tb + t) * (uint64_t)g.n_out + nb + n] = v;
                } else {
                    if (g.gate) v = v * gate[m];
                    if (g.res) v = v + res[m];
                    i8_store(g.y, g.ytype, (uint64_t)(tb + t) * g.ldy + nb + n, v);
                }
            }
        }
        wave_lds_sync();
    }
}

// The tiles: wavefronts over weight rows, tokens and K, each one's 32-row and 32-token tiles, the ring's stages (0: WIDE);
// then what a workgroup takes beside K and a 1024 values of K, in tenths of a microsecond (a fit, half_gemm.hip).
#define SYN_HALF_TILES(X)             \
    X(0, 4, 2, 1, 2, 4, 0, 45, 213)   \
    X(1, 2, 2, 1, 2, 2, 0, 24, 80)    \
    X(2, 1, 2, 2, 2, 2, 4, 17, 58)    \
    X(3, 1, 1, 4, 2, 2, 4, 20, 33)    \
    X(4, 1, 1, 4, 2, 1, 4, 15, 24)    \
    X(5, 1, 1, 4, 1, 1, 4, 9, 18)

template <class C, int WTY, int OT>
static void launch_as(const HalfArgs& a, hipStream_t stream) {
    const int tw = (a.n_out + C::BM - 1) / C::BM, tt = (a.T + C::BN - 1) / C::BN;
    static std::atomic<uint64_t> said{0};
    i8_allow_lds((const void*)k_half_gemm<C, WTY, OT>, C::LDS, said);
    hipLaunchKernelGGL((k_half_gemm<C, WTY, OT>), dim3((uint32_t)tw * (uint32_t)tt, 1, a.splits), dim3(64 * C::NW), C::LDS,
                       stream, a, tw, tt);
}
template <class C, int WTY>
static void launch_out(const HalfArgs& a, hipStream_t stream) {
    if (a.splits > 1)
        launch_as<C, WTY, OUT_PART>(a, stream);
    else if (a.ytype == T_F32)
        launch_as<C, WTY, OUT_F32>(a, stream);
    else
        launch_as<C, WTY, OUT_16>(a, stream);
}

template <int WTY>
static void launch_half_tile(int tile, const HalfArgs& a, hipStream_t stream) {
#define SYN_HALF_CASE(id, wm, wn, wk, mt, nt, ring, base, k) \
    case id: launch_out<HalfTile<wm, wn, wk, mt, nt, ring>, WTY>(a, stream); break;
    switch (tile) { SYN_HALF_TILES(SYN_HALF_CASE) }
#undef SYN_HALF_CASE
}

}  // namespace syn
