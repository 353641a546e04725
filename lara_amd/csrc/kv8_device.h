// Rows of the E4M3 cache: one row (the D values of a token of a kv head, K and V apart) is D codes and one scale
// byte, value = code * 2^(byte - 127).
//
// Writing a row: a = its largest finite |x| (at most kKv8Top); byte = the least one with 448 * 2^(byte - 127) >= a (1 at
// the least); code = x * 2^(127 - byte) rounded to nearest even; infinities and NaN become NaN.  A power of two costs
// no accuracy against a / 448 (the codes are floating point themselves), makes the division exact, so that a value is
// rounded once (half a step: 2^-4 of it, or 2^-10 * 2^(byte - 127) below 2^-6 * 2^(byte - 127)), and the value read
// back exact in bf16.
#pragma once

#include "gqa_internal.h"

namespace lara {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// The largest magnitude a row holds, 1.875 * 2^127: beyond it the nearest code stands for 2^128.
constexpr uint32_t kKv8TopBits = 0x7F700000u;

template <int CTRL>
__device__ __forceinline__ uint32_t max_dpp(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return o > v ? o : v;
}

// Maximum over the LANES (8 or 16) lanes of a row, in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    static_assert(LANES == 8 || LANES == 16, "a row of D values takes D / 8 lanes");
    v = max_dpp<0xB1>(v);   // quad_perm [1, 0, 3, 2]
    v = max_dpp<0x4E>(v);   // quad_perm [2, 3, 0, 1]
    v = max_dpp<0x141>(v);  // row_half_mirror
    if constexpr (LANES == 16) v = max_dpp<0x140>(v);  // row_mirror
    return v;
}

// Quantises a row held by LANES lanes, 8 values each: a lane's 8 codes, and the row's scale byte in every lane.
template <int LANES>
__device__ __forceinline__ u32x2 kv8_quantise(const float (&x)[8], uint32_t* scale_byte) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t mag = __float_as_uint(x[i]) & 0x7FFFFFFFu;
        const uint32_t held = mag > kKv8TopBits ? kKv8TopBits : mag;
        if (mag < 0x7F800000u && held > top) top = held;
    }
    top = row_max<LANES>(top);
    const int exponent = (int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);  // (1.75 * 2^8 = 448)
    const uint32_t byte = exponent < 1 ? 1u : (uint32_t)exponent;
    *scale_byte = byte;
    const float inverse = __uint_as_float((254u - byte) << 23);
    const float limit = __uint_as_float(kKv8TopBits);
    float c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool finite = (__float_as_uint(x[i]) & 0x7F800000u) != 0x7F800000u;
        c[i] = finite ? __builtin_amdgcn_fmed3f(x[i], -limit, limit) * inverse : __uint_as_float(0x7FC00000u);
    }
    u32x2 out;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * w], c[4 * w + 1], 0, false);
        v = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * w + 2], c[4 * w + 3], v, true);
        out[w] = (uint32_t)v;
    }
    return out;
}

// Eight bf16 words as fp32.
__device__ __forceinline__ void unpack_bf16x8(const u32x4& w, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(w[j] << 16);
        x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
}

// The value of a scale byte (0, the byte of rows never written, stands for 0: their codes are 0 too).
__device__ __forceinline__ float kv8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// Row index of token t of (b, kv head h), or -1 where its page is unmapped.
__device__ __forceinline__ int64_t kv8_row(const Kv8Cache& c, int b, int h, int t) {
    if (c.block_table != nullptr)
        return paged_row(c.block_table + (size_t)b * c.max_pages, c.page_shift, c.n_kv_heads, h, t);
    return ((int64_t)b * c.n_kv_heads + h) * c.l_cap + t;
}

}  // namespace
}  // namespace lara
