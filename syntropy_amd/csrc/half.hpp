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
// gelu is v Phi(v) with Phi(-x) = erfc(x / sqrt 2) / 2, which keeps its relative accuracy where v is far below 0 and
// 1 + erf would cancel.  With t = 1 / (1 + 0.4 x / sqrt 2) the logarithm of erfc(x / sqrt 2) exp(x^2 / 2) / t is
// smooth in t: a polynomial of degree 8, a minimax fit over x from 0 to 17 (9.1e-8; in F32 4.3e-7 of the result, no
// branches).  (With the library's erfc, some 150 instructions on both sides of a branch, 5003 x 2011 at 333 tokens took
// 9 us more than without an activation.)
SYN_DEV float half_gelu(float v) {
    constexpr double C = -0.72134752044448170368;  // -log2(e) / 2
    constexpr float HI = (float)C, LO = (float)(C - (double)HI);
    const float x = fminf(__builtin_fabsf(v), 20.0f);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(x, 0.28284271247461900976f, 1.0f));
    float q = -0.30159053206443787f;
    q = __builtin_fmaf(q, t, 1.345345377922058f);
    q = __builtin_fmaf(q, t, -2.168454647064209f);
    q = __builtin_fmaf(q, t, 1.4710724353790283f);
    q = __builtin_fmaf(q, t, -0.6613202691078186f);
    q = __builtin_fmaf(q, t, 0.44308316707611084f);
    q = __builtin_fmaf(q, t, 0.5741007924079895f);
    q = __builtin_fmaf(q, t, 1.4455450773239136f);
    q = __builtin_fmaf(q, t, -2.1477816104888916f);
    const float s = x * x, sr = __builtin_fmaf(x, x, -s);
    const float e = s * HI, er = __builtin_fmaf(sr, HI, __builtin_fmaf(s, LO, __builtin_fmaf(s, HI, -e)));
    const float n = __builtin_rintf(e);
    const float tail = __builtin_ldexpf(0.5f * x * t * __builtin_amdgcn_exp2f((e - n) + (q + er)), (int)n);
    return v < 0.0f ? (v - v) - tail : v - tail;  // (a NaN at -infinity, as the formula)
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
template <int ACT>
SYN_DEV float half_act(float v) {
    if constexpr (ACT == HALF_RELU) return v < 0.0f ? 0.0f : v;  // (a NaN stays one)
    if constexpr (ACT == HALF_SILU) return i8_silu(v);
    if constexpr (ACT == HALF_GELU) return half_gelu(v);
    if constexpr (ACT == HALF_GELU_TANH) return half_gelu_tanh(v);
    return v;
}
// f(the activation's constant) of a uniform `act`.
template <class F>
SYN_DEV void half_act_of(int act, F&& f) {
    switch (act) {
        case HALF_RELU: return f(std::integral_constant<int, HALF_RELU>{});
        case HALF_SILU: return f(std::integral_constant<int, HALF_SILU>{});
        case HALF_GELU: return f(std::integral_constant<int, HALF_GELU>{});
        case HALF_GELU_TANH: return f(std::integral_constant<int, HALF_GELU_TANH>{});
        default: return;
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

// N (4 or 8) values that are all there as they lie in memory, at most 16 bytes, to be unpacked when they are used.
template <int N>
struct HalfRaw {
    uint32_t w[4];
};
template <int N>
SYN_DEV void half_fetch(const void* p, int ty, uint64_t i, HalfRaw<N>& raw) {
    if (N == 4 && ty == T_F32)
        __builtin_memcpy(raw.w, (const float*)p + i, 16);
    else
        __builtin_memcpy(raw.w, (const uint16_t*)p + i, 2 * N);
}
template <int N>
SYN_DEV void half_unpack(int ty, const HalfRaw<N>& raw, float (&v)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t b = raw.w[j / 2] >> (16 * (j & 1)) & 0xFFFFu;
        v[j] = ty == T_F16 ? f16_to_f32(b) : u2f(b << 16);
        if constexpr (N == 4) v[j] = ty == T_F32 ? u2f(raw.w[j]) : v[j];
    }
}

// Four outputs (the first `in` of them) of token t from their sums, with what the epilogue reads:
// y = act(sum + bias) gate + residual in F32, rounded once.
struct HalfRest {
    float bias[4], gate[4], res[4];
};
SYN_DEV HalfRest half_rest(const HalfArgs& g, int t, int64_t n, int in) {
    HalfRest r{};
    if (g.bias) half_load<4>(g.bias, T_F32, (uint64_t)n, in, r.bias);
    if (g.gate) half_load<4>(g.gate, g.gtype, (uint64_t)t * g.ldg + n, in, r.gate);
    if (g.res) half_load<4>(g.res, g.rtype, (uint64_t)t * g.ldr + n, in, r.res);
    return r;
}
SYN_DEV void half_emit(const HalfArgs& g, int t, int64_t n, int in, float (&v)[4], const HalfRest& r) {
    if (g.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = v[e] + r.bias[e];
    }
    half_act_of(g.act, [&](auto act) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = half_act<decltype(act)::value>(v[e]);
    });
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (e >= in) break;
        if (g.gate) v[e] = v[e] * r.gate[e];
        if (g.res) v[e] = v[e] + r.res[e];
        i8_store(g.y, g.ytype, (uint64_t)t * g.ldy + n + e, v[e]);
    }
}

// half_few.hip: up to 8 tokens, weights straight to registers; x at any address
bool half_few_fits(int T);
void launch_half_few(const HalfArgs& a, hipStream_t stream);
// half_gemm.hip: tiles through LDS, K in one part or several; x's rows are whole pairs of lines on 16 bytes
struct HalfPick {
    int tile, splits;
};
HalfPick half_gemm_pick(int n_out, int k, int T);
bool half_gemm_reaches(int tile, const HalfArgs& a);
void launch_half_gemm(int tile, const HalfArgs& a, hipStream_t stream);
void launch_half_gemm_f16(int tile, const HalfArgs& a, hipStream_t stream);
void launch_half_gemm_bf16(int tile, const HalfArgs& a, hipStream_t stream);
// half.hip
// lines: x's rows are whole pairs of lines on 16 bytes; else they are copied into the workspace where they have to be.
uint64_t half_ws_bytes(int n_out, int k, int T, bool lines);
void launch_half_gemv(const HalfArgs& a, bool lines, uint8_t* ws, hipStream_t stream);

}  // namespace syn
