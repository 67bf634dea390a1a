// Products over int8 weights with a scale a channel (output row), the activations quantized to int8 with
// a scale a token: shared geometry and device helpers.
#pragma once

#include <atomic>
#include <type_traits>

#include "common.hpp"

namespace syn {

typedef int i8x16 __attribute__((ext_vector_type(4)));  // sixteen int8 codes
typedef int i32x16 __attribute__((ext_vector_type(16)));

// The tokens' codes are held in rows of whole pairs of 128-byte lines, zeros behind the last value, so that
// what a kernel reads of a weight row past its end is multiplied by zero.
constexpr int I8_LINE = 128;
SYN_HD inline uint64_t i8_padded(uint64_t k) { return align_up(k, 2 * I8_LINE); }
// |sum| <= 128 * 127 * k stays below 2^31.
constexpr uint32_t I8_MAX_K = 131072;

// A workspace: codes [rows][padded k], then F32 scales [rows], then the partial sums of a split K.
struct I8Act {
    uint64_t scales, partial;
};
SYN_HD inline I8Act i8_act_layout(uint64_t rows, uint64_t k) {
    I8Act a;
    a.scales = align_up(rows * i8_padded(k), 256);
    a.partial = a.scales + 4 * align_up(rows, 256);  // (a tile reads the scales of its last rows' places too)
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

// Eight values from i on of a row of k (zeros past its end), at any alignment.
template <int TY>
SYN_DEV void i8_load8(const uint8_t* xr, int i, int k, float (&v)[8]) {
    if (i + 8 <= k) {
        if constexpr (TY == T_F32) {
            __builtin_memcpy(v, xr + 4 * (int64_t)i, 32);
        } else {
            uint32_t h[4];
            __builtin_memcpy(h, xr + 2 * (int64_t)i, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t b = h[j / 2] >> (16 * (j & 1)) & 0xFFFFu;
                v[j] = TY == T_F16 ? f16_to_f32(b) : u2f(b << 16);
            }
        }
    } else if (i < k) {  // (loads at places that are there, all in flight: a branch around each would wait for the one before)
        uint32_t h[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int in = i + j < k ? i + j : k - 1;
            h[j] = TY == T_F32 ? ((const uint32_t*)xr)[in] : ((const uint16_t*)xr)[in];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float f = TY == T_F32 ? u2f(h[j]) : TY == T_F16 ? f16_to_f32(h[j]) : u2f(h[j] << 16);
            v[j] = i + j < k ? f : 0.0f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    }
}
// BF16 by round to nearest even, a NaN kept one.
SYN_DEV uint32_t bf16_bits(float v) {
    const uint32_t u = f2u(v);
    return v != v ? 0x7FC0u : (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
template <int TY>
SYN_DEV uint32_t i8_half2(float a, float b) {
    if constexpr (TY == T_F16)
        return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)a) | (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)b) << 16;
    else
        return bf16_bits(a) | bf16_bits(b) << 16;
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
// The largest magnitude's bits of eight values and m.
SYN_DEV uint32_t i8_max8(const float (&v)[8], uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t b = f2u(v[j]) & 0x7FFFFFFFu;
        m = m > b ? m : b;
    }
    return m;
}
// Their codes.  (Where inv is 0 the codes are 0, whatever the value: an infinity times 0 is a NaN.)
SYN_DEV uint2 i8_codes8(const float (&v)[8], float inv) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j / 4] |= ((uint32_t)(int)__builtin_rintf(v[j] * inv) & 0xFFu) << (8 * (j & 3));
    return inv == 0.0f ? uint2{0, 0} : uint2{w[0], w[1]};
}

// An output from its exact sum: RN(RN(RN(S) sx) sw), the bias added.  |S| may pass 2^24, so the first
// rounding is the conversion's.
SYN_DEV float i8_value(int sum, float sx, float sw) { return ((float)sum * sx) * sw; }

// silu(g) = g / (1 + exp(-g)) within 2^-21 of its value, to F32's least subnormal: exp(-g) as 2^t of the rounded
// product t = -g log2(e) and a factor for what that leaves, the rounding and what F32's log2(e) lacks (1.9e-8:
// at g = -88 ten steps of the result).  Below -80 the power is taken 2^32 times less, beside which the 1 still
// counts for nothing, and the quotient brought back by one product: v_rcp_f32 keeps few bits of a subnormal
// result, and a quotient that is one rounds once.  Below -111 the power is infinite and the quotient 0 (a value
// below 2^-150).  An infinite or NaN g is met in the product with g.  (14336 x 4096 gated at 1024 tokens 138.7 us;
// 137.2 with neither the rest of log2(e) nor the values below -88.)
SYN_DEV float i8_silu(float g) {
    constexpr float LOG2E = 1.44269504088896340736f, LOG2E_REST = (float)(1.44269504088896340736 - (double)LOG2E);
    const bool far = g < -80.0f;
    const float gc = __builtin_amdgcn_fmed3f(g, -180.0f, 100.0f);
    const float t = gc * -LOG2E;
    const float r = __builtin_fmaf(gc, -LOG2E_REST, __builtin_fmaf(gc, -LOG2E, -t));
    const float e = __builtin_amdgcn_exp2f(t + (far ? -32.0f : 0.0f)) * __builtin_fmaf(r, 0.69314718055994530942f, 1.0f);
    return g * __builtin_amdgcn_rcpf(1.0f + e) * (far ? 0x1p-32f : 1.0f);
}

// Workgroups go to the 8 XCDs in turn.  Each XCD takes a run of neighbouring tiles, token tiles first within
// groups of 8, so that what runs on it at once shares its weight rows and tokens in its L2.
SYN_DEV void i8_tile_of(int id, int tiles_w, int tiles_t, int& tw, int& tt) {
    const int total = tiles_w * tiles_t, each = total / 8, rest = total % 8, x = id & 7;
    int l = x * each + (x < rest ? x : rest) + id / 8;
    const int group = 8 * tiles_w, gi = l / group, t8 = gi * 8;
    const int in = tiles_t - t8 < 8 ? tiles_t - t8 : 8;
    l -= gi * group;
    tt = t8 + l % in;
    tw = l / in;
}

// Before a launch of `kernel`: allows it so much dynamic LDS on the current device, whose attribute the limit is;
// `said`, the kernel's own, holds a bit for each device that it was said to.  A refusal shows as the launch's error.
inline void i8_allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& said) {
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess) return;
    const uint64_t bit = device < 64 ? 1ull << device : 0;  // (a device past those is told every time)
    if (said.load(std::memory_order_acquire) & bit) return;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess)
        said.fetch_or(bit, std::memory_order_release);
}

void launch_i8_quantize(int xtype, const void* x, uint64_t ldx, int rows, int k, int8_t* codes, uint64_t ldc,
                        float* scales, hipStream_t stream);
// int8_few.hip: up to 16 tokens, weights straight to registers
bool i8_few_fits(int rows_w, int T);
bool i8_few_fused(int rows_w, int k, int T);  // the kernel quantizes the rows itself
void launch_i8_few(const I8Args& a, hipStream_t stream);
// int8_gemm.hip: tiles through LDS, K in one part or several
struct I8Pick {
    int tile, splits;
};
I8Pick i8_gemm_pick(int rows_w, int k, int T);
bool i8_gemm_reaches(int tile, const I8Args& a);
void launch_i8_gemm(int tile, const I8Args& a, hipStream_t stream);
// int8.hip
int i8_splits(int rows_w, int k, int T);
bool i8_fused(int rows_w, int k, int T);
void launch_i8_gemv(const I8Args& a, hipStream_t stream);

}  // namespace syn
