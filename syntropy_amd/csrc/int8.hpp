// Products over int8 weights with a scale a channel (output row), the activations quantized to int8 with
// a scale a token: shared geometry and device helpers.
#pragma once

#include "common.hpp"

namespace syn {

typedef int i8x16 __attribute__((ext_vector_type(4)));  // sixteen int8 codes
typedef int i32x16 __attribute__((ext_vector_type(16)));

// The tokens' codes are held in rows of whole 128-byte lines, zeros behind the last value, so that what
// a kernel reads of a weight row past its end is multiplied by zero.
constexpr int I8_LINE = 128;
SYN_HD inline uint64_t i8_padded(uint64_t k) { return align_up(k, I8_LINE); }
// |sum| <= 128 * 127 * k stays below 2^31.
constexpr uint32_t I8_MAX_K = 131072;

// A workspace: codes [rows][padded k], then F32 scales [rows], then the partial sums of a split K.
struct I8Act {
    uint64_t scales, partial;
};
SYN_HD inline I8Act i8_act_layout(uint64_t rows, uint64_t k) {
    I8Act a;
    a.scales = align_up(rows * i8_padded(k), 256);
    a.partial = align_up(a.scales + 4 * rows, 256);
    return a;
}

struct I8Args {
    const int8_t* w;       // [n_out or 2 n_out][k], rows ldw bytes apart, each on 16 bytes
    uint64_t ldw;
    const float* ws;       // a scale a row of w
    const float* bias;     // or null
    int n_out, k;
    const int8_t* xq;      // [T][padded k]
    const float* xs;       // [T]
    const void* x;         // the rows before quantization, for the kernel that quantizes them itself
    uint64_t ldx;          // in values
    int xtype;
    int T;
    void* y;               // [T][n_out], rows ldy values apart
    uint64_t ldy;
    int ytype;
    int* partial;          // [splits][T][rows of w] where K is split over workgroups
    int splits;
    int gated;             // w is [gate; up]: y = silu(gate) * up
};

SYN_DEV float i8_load(const void* x, int ty, uint64_t i) {
    if (ty == T_F32) return ((const float*)x)[i];
    const uint32_t h = ((const uint16_t*)x)[i];
    return ty == T_F16 ? f16_to_f32(h) : u2f(h << 16);
}
// BF16 by round to nearest even, a NaN kept one.
SYN_DEV uint32_t bf16_bits(float v) {
    const uint32_t u = f2u(v);
    return v != v ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
SYN_DEV void i8_store(void* y, int ty, uint64_t i, float v) {
    if (ty == T_F32)
        ((float*)y)[i] = v;
    else if (ty == T_F16)
        ((_Float16*)y)[i] = (_Float16)v;
    else
        ((uint16_t*)y)[i] = (uint16_t)bf16_bits(v);
}

// A token's scale and the factor of its codes from its largest magnitude's bits: s = a / 127, codes
// rint(x / s) by the rounded inverse (0 where s or the inverse says nothing); a NaN or an infinity in the
// row gives the scale NaN and codes 0, so that every output of the row is NaN.
struct I8Scale {
    float s, inv;
};
SYN_DEV I8Scale i8_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return {__builtin_nanf(""), 0.0f};
    const float s = div127(u2f(amax_bits));
    const float inv = s != 0.0f ? recip_rn(s) : 0.0f;
    return {s, finite_f(inv) ? inv : 0.0f};
}
// (a row with a NaN or an infinity: v inv may be a NaN, whose conversion is 0; an infinity's is not, so
// the factor's sign says nothing and the code is zeroed by the caller through `inv` = 0)
SYN_DEV int i8_code(float v, float inv) {
    return inv == 0.0f ? 0 : (int)__builtin_rintf(v * inv);
}

// An output from its exact sum: RN(RN(RN(S) sx) sw), the bias added.  |S| may pass 2^24, so the first
// rounding is the conversion's.
SYN_DEV float i8_value(int sum, float sx, float sw) { return ((float)sum * sx) * sw; }

void launch_i8_quantize(int xtype, const void* x, uint64_t ldx, int rows, int k, int8_t* codes, uint64_t ldc,
                        float* scales, hipStream_t stream);
int i8_splits(int rows_w, int k, int T, int gated);
void launch_i8_gemv(const I8Args& a, hipStream_t stream);
bool i8_fused(int rows_w, int k, int T, int gated);

}  // namespace syn
