// The half-precision product at few tokens (one to eight): bound by reading the weights once from HBM.
//
// v_mfma_f32_16x16x32 multiplies 16 rows by 16 columns over 32 values, four lanes a row of 8 values each.  Its rows
// are taken as 8 weight rows x the two halves of a 128-byte line and its columns as 8 tokens x the same halves: where
// a row's half is a column's, the product is one that is wanted (the other quarters are not looked at).  So a lane
// loads 16 bytes of a weight row straight to the registers that the instruction reads, and an instruction loads
// whole lines of 8 rows.  No other wavefront reads them, so LDS would only be a detour.
// The eight wavefronts of a workgroup share 8 RT rows and take turns at K, U lines at a time, two turns in flight;
// their sums meet in LDS, always in the same order.  The tokens' values of a turn are loaded with its weights (loads
// return in order), what the epilogue reads before them all.
#include "half.hpp"
#include "kernels.hpp"

namespace syn {

// LINES: x's rows are whole pairs of lines on 16 bytes.
template <int WTY, int RT, int U, int NW, int LINES>
__global__ __launch_bounds__(64 * NW, 6) void k_half_few(HalfArgs g) {
    static_assert(RT <= 4, "the outputs of one wavefront");
    __shared__ f32x4 red[NW][RT][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 7;                                       // weight row, and token, of 8
    const int piece = 8 * (4 * ((lane >> 3) & 1) + (lane >> 4));  // of a line, in values
    const int lines = (int)half_padded(g.k) / 64;
    const int t0 = (int)blockIdx.y * 8;
    const int nt = g.T - t0 < 8 ? g.T - t0 : 8;
    const int64_t n0 = (int64_t)blockIdx.x * 8 * RT;
    const uint16_t* wr[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int64_t n = n0 + 8 * i + c;
        wr[i] = g.w + (uint64_t)(n < g.n_out ? n : g.n_out - 1) * g.ldw + piece;
    }
    const uint16_t* xr = g.x + (uint64_t)(t0 + c) * g.ldx;
    constexpr int TURN = U * NW;  // lines
    struct Turn {
        i8x16 w[U][RT], x[U];
    };
    auto load = [&](int s, Turn& to) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= lines) break;  // uniform
#pragma unroll
            for (int i = 0; i < RT; ++i)
                to.w[u][i] = __builtin_nontemporal_load(reinterpret_cast<const i8x16*>(wr[i] + 64 * (s + u)));
            to.x[u] = i8x16{0, 0, 0, 0};
            if (c >= nt) continue;
            const int at = 64 * (s + u) + piece;
            const uint16_t* from = xr + at;
            if constexpr (LINES) {
                to.x[u] = *reinterpret_cast<const i8x16*>(from);
            } else if (at + 8 <= g.k) {
                __builtin_memcpy(&to.x[u], from, 16);
            } else if (at < g.k) {
                uint32_t h[4] = {};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (at + e < g.k) h[e / 2] |= (uint32_t)from[e] << (16 * (e & 1));
                to.x[u] = i8x16{(int)h[0], (int)h[1], (int)h[2], (int)h[3]};
            }
        }
    };
    // the outputs of lane l: tile l / 16, rows 4 (l / 8 & 1) .. + 3, token l & 7; by the first wavefront
    const int tile = lane >> 4, half = (lane >> 3) & 1;
    const int64_t n = n0 + 8 * tile + 4 * half;
    const int in = wave == 0 && tile < RT && c < nt ? (g.n_out - n < 4 ? (int)(g.n_out - n) : 4) : 0;
    HalfRest rest{};
    if (in > 0) rest = half_rest(g, t0 + c, n, in);
    Turn cur, nxt;
    int s = wave * U;
    load(s, cur);
    load(s + TURN, nxt);
    f32x4 acc[RT] = {};
    auto product = [&](int s, const Turn& o) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s + u >= lines) break;  // uniform
#pragma unroll
            for (int i = 0; i < RT; ++i) acc[i] = half_mfma16<WTY>(o.w[u][i], o.x[u], acc[i]);
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
#pragma unroll
    for (int i = 0; i < RT; ++i) red[wave][i][lane] = acc[i];
    __syncthreads();
    if (in <= 0) return;
    f32x4 sum = {};
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += red[w][tile][16 * half + c] + red[w][tile][16 * half + 40 + c];
    float v[4] = {sum[0], sum[1], sum[2], sum[3]};
    half_emit(g, t0 + c, n, in, v, rest);
}

// Against the tiles (BF16, us, at 8 rows): 4096 x 4096 9.2 and 10.5, 14336 x 4096 25.0 and 23.9, 4096 x 14336 24.1 and 25.4,
// 32000 x 4096 46.9 and 54.7, 1024 x 1024 4.1 and 4.2.  At 16 rows the tokens' values weigh as much as the weights here,
// and the tiles' LDS pays: 10.6 and 10.7, 32.0 and 24.0, 29.0 and 25.5, 60.7 and 55.5, 4.6 and 4.2.
bool half_few_fits(int T) { return T <= 8; }

template <int WTY, int RT, int U, int NW>
static void launch_few(const HalfArgs& a, hipStream_t stream) {
    const dim3 grid((a.n_out + 8 * RT - 1) / (8 * RT), (a.T + 7) / 8);
    const bool lines = a.k % HALF_PAIR == 0 && (uintptr_t)a.x % 16 == 0 && (a.T <= 1 || a.ldx % 8 == 0);
    if (lines)
        hipLaunchKernelGGL((k_half_few<WTY, RT, U, NW, 1>), grid, dim3(64 * NW), 0, stream, a);
    else
        hipLaunchKernelGGL((k_half_few<WTY, RT, U, NW, 0>), grid, dim3(64 * NW), 0, stream, a);
}
// 16 weight rows a workgroup read each token's values for twice as many products as 8, and leave half as many workgroups:
// taken from three tokens on where their last round over the 256 CUs is full enough (4096 x 4096 at 8 tokens 9.2 us and
// 10.5, 32000 x 4096 46.9 and 59.6; 6144 x 4096 at 4, one round and a half, 14.0 and 12.5, 2048 x 8192 12.3 and 9.5).
template <int WTY>
static void launch_some(const HalfArgs& a, hipStream_t stream) {
    const int64_t wgs = ((int64_t)a.n_out + 15) / 16, rounds = (wgs + 255) / 256;
    if (a.T > 2 && 5 * wgs >= 4 * 256 * rounds)
        launch_few<WTY, 2, 1, 8>(a, stream);
    else
        launch_few<WTY, 1, 2, 8>(a, stream);
}

// (any number of tokens, for rows that a tile's offsets do not reach: as many a launch as a grid holds)
void launch_half_few(const HalfArgs& a, hipStream_t stream) {
    constexpr int MOST = 1 << 18;
    auto at = [](const void* p, int ty, uint64_t ld, int t) {
        return p ? (const uint8_t*)p + (uint64_t)t * ld * (ty == T_F32 ? 4 : 2) : nullptr;
    };
    for (int t = 0; t < a.T; t += MOST) {
        HalfArgs g = a;
        g.T = a.T - t < MOST ? a.T - t : MOST;
        g.x = a.x + (uint64_t)t * a.ldx;
        g.gate = at(a.gate, a.gtype, a.ldg, t);
        g.res = at(a.res, a.rtype, a.ldr, t);
        g.y = (void*)at(a.y, a.ytype, a.ldy, t);
        a.wtype == T_F16 ? launch_some<T_F16>(g, stream) : launch_some<T_BF16>(g, stream);
    }
}

}  // namespace syn
