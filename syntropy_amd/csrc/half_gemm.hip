// Which tile the half-precision product takes (half_gemm.hpp), and its launch.
#include "half_gemm.hpp"

namespace syn {

struct TileOf {
    int m, n;           // weight rows, tokens
    float base, per_k;  // microseconds a workgroup, and a value of K
};
#define SYN_HALF_TILE(id, wm, wn, wk, mt, nt, ring, base, k) {32 * wm * mt, 32 * wn * nt, 0.1f * base, 0.1f * k / 1024},
static const TileOf TILES[] = {SYN_HALF_TILES(SYN_HALF_TILE)};
#undef SYN_HALF_TILE

// The tile and the parts of K that are estimated to take least: rounds of 256 workgroups, the last one's faster the fewer
// there are in it, beside what the weights take from HBM (5.6 TB/s at most, 92 GB/s a workgroup, and part of a reading
// more for every further tile of tokens): the longer of the two and a quarter of the other; K in parts costs the
// fold's launch and its partial sums' writing and reading.  The constants are a fit to 500 measured calls; of 51 matrices
// and row counts 43 run on the fastest choice, 6 within 8 % of it, two at 11 and 14.  Large tiles read less from L2
// for an output, small ones fill the chip: 4096 x 4096 at 512 tokens takes 27 us in 256 tiles of 64 x 128 and 37 in
// 128 of 128 x 128, at 32 tokens 11.5 in 128 of 32 x 32 and 12.7 in 64 of 64 x 32 by four parts of K; 14336 x 4096 at 2048
// tokens 202 in 448 of 256 x 256 and 232 in 1792 of 128 x 128.
HalfPick half_gemm_pick(int n_out, int k, int T) {
    constexpr float LAUNCH = 2.3f, FOLD = 3.0f;                     // us
    constexpr float HBM = 5.6e6f, EACH = 9.2e4f, SUMS = 5.4e6f;     // bytes a us
    const int kp = (int)half_padded(k);
    HalfPick best{0, 1};
    float least = 0.0f;
    for (int i = 0; i < (int)(sizeof TILES / sizeof TILES[0]); ++i) {
        const TileOf& t = TILES[i];
        const int64_t tw = (n_out + t.m - 1) / t.m, tt = (T + t.n - 1) / t.n;
        const float bytes = 2.0f * (float)n_out * (float)k * (tt < 4 ? 0.6f + 0.4f * (float)tt : 2.0f);
        for (int s = 1; s <= 8; s = s < 4 ? s + 1 : s + 2) {
            const int64_t wgs = tw * tt * s, rounds = (wgs + 255) / 256;
            if (s > 1 && (kp < 512 * s || wgs > 256)) break;  // (a part has four stages and more)
            const float last = (float)(wgs - 256 * (rounds - 1)) / 256.0f, turns = (float)rounds - 0.26f + 0.26f * last;
            const float work = (float)rounds * t.base + turns * t.per_k * (float)kp / (float)s;
            const float rate = EACH * (float)wgs < HBM ? EACH * (float)wgs : HBM;
            const float read = bytes / rate;
            float us = LAUNCH + (work > read ? work + 0.25f * read : read + 0.25f * work);  // (they overlap in part)
            if (s > 1) us += FOLD + 8.0f * (float)s * (float)T * (float)n_out / SUMS;
            if (least == 0.0f || us < least) {
                least = us;
                best = HalfPick{i, s};
            }
        }
    }
    return best;
}

bool half_gemm_reaches(int tile, const HalfArgs& a) {
    return 2 * (uint64_t)TILES[tile].m * a.ldw < (1ull << 31) && 2 * (uint64_t)TILES[tile].n * a.ldx < (1ull << 31);
}

void launch_half_gemm(int tile, const HalfArgs& a, hipStream_t stream) {
    a.wtype == T_F16 ? launch_half_gemm_f16(tile, a, stream) : launch_half_gemm_bf16(tile, a, stream);
}

}  // namespace syn
