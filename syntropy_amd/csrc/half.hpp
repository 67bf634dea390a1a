// Products over F16 or BF16 weights with an epilogue: shared arguments and device helpers.
#pragma once

#include "int8.hpp"

namespace syn {

enum HalfAct { HALF_NONE = 0, HALF_RELU, HALF_SILU, HALF_GELU, HALF_GELU_TANH };

// Rows of weights are followed by zeros up to whole pairs of 128-byte lines, and so are those of a copy of x.
constexpr int HALF_PAIR = 128;  // values
SYN_HD inline uint64_t half_padded(uint64_t k) { return align_up(k, HALF_PAIR); }
constexpr uint32_t HALF_MAX_K = 1 << 20;

struct HalfArgs {
    int wtype;             // of w and x
    const uint16_t* w;     // [n_out][k], rows ldw values apart, each on 16 bytes
    uint64_t ldw;
    const float* bias;     // [n_out] or null
    int n_out, k;
    const uint16_t* x;     // [T][k], rows ldx values apart
    uint64_t ldx;
    int T;
    int act;
    const void* gate;      // [T][n_out] or null
    uint64_t ldg;
    int gtype;
    const void* res;       // [T][n_out] or null
    uint64_t ldr;
    int rtype;
    void* y;               // [T][n_out], rows ldy values apart
    uint64_t ldy;
    int ytype;
    float* partial;        // [splits][T][n_out] where K is split over workgroups
    int splits;
};

// The activation of an F32 sum, each within about 2^-20 of its value where that is no subnormal: the argument of
// each exponential is carried in two parts, since its rounding (2^-24 of up to 80) would be the result's error.
// gelu is v Phi(v) = v erfc(-v / sqrt 2) / 2, which keeps its relative accuracy where v is far below 0 and
// 1 + erf would cancel; d erfc(a) is about -2 a erfc(a) there.  The tanh form of it is v / (1 + exp(-2 z)), the
// value of v (1 + tanh z) / 2 without its cancellation, 2 z = v (c1 + c2 v^2).
SYN_DEV float half_gelu(float v) {
    constexpr double C = -0.70710678118654752440;
    constexpr float HI = (float)C, LO = (float)(C - (double)HI);
    const float a = v * HI, rest = __builtin_fmaf(v, LO, __builtin_fmaf(v, HI, -a));
    return 0.5f * v * (erfcf(a) * (a > 1.0f && a < 12.0f ? __builtin_fmaf(-2.0f * a, rest, 1.0f) : 1.0f));
}
SYN_DEV float half_gelu_tanh(float v) {
    constexpr double C1 = 1.5957691216057307117, C2 = C1 * 0.044715;
    constexpr float A1 = (float)C1, B1 = (float)(C1 - (double)A1), A2 = (float)C2, B2 = (float)(C2 - (double)A2);
    if (!(__builtin_fabsf(v) < 32.0f)) return v > 0.0f ? v : v * 0.0f;  // (a NaN and -infinity give a NaN)
    const float s = v * v, sr = __builtin_fmaf(v, v, -s);
    const float q = A2 * s, p = q + A1, back = p - q;  // (p's rounding by both summands)
    const float pr = ((q - (p - back)) + (A1 - back)) + __builtin_fmaf(A2, s, -q) + __builtin_fmaf(A2, sr, __builtin_fmaf(B2, s, B1));
    const float z = v * p, zr = __builtin_fmaf(v, pr, __builtin_fmaf(v, p, -z));
    return i8_times_sigmoid(v, z, zr * 1.44269504088896340736f);
}
SYN_DEV float half_act(int act, float v) {
    switch (act) {
        case HALF_RELU: return v < 0.0f ? 0.0f : v;  // (a NaN stays one)
        case HALF_SILU: return i8_silu(v);
        case HALF_GELU: return half_gelu(v);
        case HALF_GELU_TANH: return half_gelu_tanh(v);
        default: return v;
    }
}

SYN_DEV float half_at(const void* p, int ty, uint64_t i) {
    if (ty == T_F32) return ((const float*)p)[i];
    const uint32_t h = ((const uint16_t*)p)[i];
    return ty == T_F16 ? f16_to_f32(h) : u2f(h << 16);
}

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// Eight values of each of 32 (16) rows and columns a lane.
template <int WTY>
SYN_DEV f32x16 half_mfma32(i8x16 a, i8x16 b, f32x16 c) {
    if constexpr (WTY == T_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <int WTY>
SYN_DEV f32x4 half_mfma16(i8x16 a, i8x16 b, f32x4 c) {
    if constexpr (WTY == T_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// N (4 or 8) values from value i on, the first `in` of them there (the rest 0), at any value's address.
template <int N>
SYN_DEV void half_load(const void* p, int ty, uint64_t i, int in, float (&v)[N]) {
    if (in >= N) {
        if (ty == T_F32) {
            __builtin_memcpy(v, (const float*)p + i, 4 * N);
        } else {
            uint32_t h[N / 2];
            __builtin_memcpy(h, (const uint16_t*)p + i, 2 * N);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t b = h[j / 2] >> (16 * (j & 1)) & 0xFFFFu;
                v[j] = ty == T_F16 ? f16_to_f32(b) : u2f(b << 16);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = j < in ? half_at(p, ty, i + j) : 0.0f;
    }
}

// One output from its sum: y = act(sum + bias) gate + residual, in F32, rounded once.
SYN_DEV void half_emit(const HalfArgs& g, int t, int n, float v) {
    if (g.bias) v = v + g.bias[n];
    v = half_act(g.act, v);
    if (g.gate) v = v * half_at(g.gate, g.gtype, (uint64_t)t * g.ldg + n);
    if (g.res) v = v + half_at(g.res, g.rtype, (uint64_t)t * g.ldr + n);
    i8_store(g.y, g.ytype, (uint64_t)t * g.ldy + n, v);
}

// half_few.hip: up to 16 tokens, weights straight to registers; x at any address
bool half_few_fits(int n_out, int T);
void launch_half_few(const HalfArgs& a, hipStream_t stream);
// half_gemm.hip: tiles through LDS, K in one part or several; x's rows are whole pairs of lines on 16 bytes
struct HalfPick {
    int tile, splits;
};
HalfPick half_gemm_pick(int n_out, int k, int T);
bool half_gemm_reaches(int tile, const HalfArgs& a);
void launch_half_gemm(int tile, const HalfArgs& a, hipStream_t stream);
// half.hip
// lines: x's rows are whole pairs of lines on 16 bytes; else they are copied into the workspace where they have to be.
uint64_t half_ws_bytes(int n_out, int k, int T, bool lines);
void launch_half_gemv(const HalfArgs& a, bool lines, uint8_t* ws, hipStream_t stream);

}  // namespace syn
