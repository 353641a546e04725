// Norms of the query and key heads with the position rotation, into Q and the cache, in one pass.
//
// Per head row h of D values (fp32 from bf16):  y = h / sqrt(mean(h^2) + eps) * w  (w nullptr: no norm), then each pair
// (2p, 2p + 1) of y is turned by position * base^(-2p / D); V rows go as they are.  Everything is fp32 up to one rounding
// at the end: to bf16, or to a row of the E4M3 cache.  The angle and its sine and cosine are 64-bit (an fp32 angle is off
// by 2^-25 of itself: 0.03 rad at position 10^6).
//
// D / 8 lanes hold a head row, so its sum of squares (and an E4M3 row's maximum) is three or four lane exchanges, and a
// lane's four pairs are the same in every head that it takes.  A work-group is a token, so an angle is made once for all
// of its heads.
//
// Bound by memory for prompts: 2048 tokens of 32 + 16 heads of 128 (50 MB) in 8.9 us beside other launches, 5.7 TB/s (11.9
// alone); a step of 64 sequences (1.4 MB) is a launch, 4.0 / 5.0.  (Loads ahead of the angles: 14.1 us alone for those 2048,
// the waves that had waited for angles while others streamed all waiting for memory at once; sine and cosine in fp32: 0.1
// less.)
#include "kv8_device.h"

#include <math.h>

namespace lara {
namespace {

constexpr int kHeadsThreads = 256;

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}
// Sum over the LANES lanes of a row, in each of them.
template <int LANES>
__device__ __forceinline__ float row_sum(float v) {
    v = add_dpp<0xB1>(v);   // quad_perm [1, 0, 3, 2]
    v = add_dpp<0x4E>(v);   // quad_perm [2, 3, 0, 1]
    v = add_dpp<0x141>(v);  // row_half_mirror
    if constexpr (LANES == 16) v = add_dpp<0x140>(v);  // row_mirror
    return v;
}

// One work-group per token.
template <int D, bool E4M3>
__global__ __launch_bounds__(kHeadsThreads) void qk_norm_rope_kernel(HeadsArgs a) {
    constexpr int LANES = D / 8, PAIRS = D / 2;
    const int token = blockIdx.x;
    const int part = threadIdx.x % LANES;
    int b = a.b, pos = a.pos_base + token, k_pos = a.k_pos_base + token, t = a.row0 + token;
    if (a.positions != nullptr) {  // one token of each sequence
        b = token;
        pos = k_pos = a.positions[token];
        t = a.rows != nullptr ? a.rows[token] : pos;
        if (pos < 0 || t < 0 || t >= a.cache.l_max) return;  // (the whole work-group) nothing of this sequence is written
    }
    __shared__ float2 turn[2][PAIRS];
    if (a.log2_base > 0.0) {
        const int sets = k_pos != pos ? 2 : 1;
        for (int i = threadIdx.x; i < sets * PAIRS; i += kHeadsThreads) {
            const int p = i % PAIRS;
            double sd, cd;
            sincos((double)(i < PAIRS ? pos : k_pos) * exp2(-2.0 * p / D * a.log2_base), &sd, &cd);
            turn[i / PAIRS][p] = make_float2((float)cd, (float)sd);
        }
        __syncthreads();
    }
    const int heads = a.n_q_heads + 2 * a.cache.n_kv_heads;
    const u32x4* const src = reinterpret_cast<const u32x4*>(a.x + (size_t)token * a.ld);
    for (int i = threadIdx.x; i < heads * LANES; i += kHeadsThreads) {  // (a row's lanes stay together)
        const int head = i / LANES;
        const bool is_q = head < a.n_q_heads, is_k = !is_q && head < a.n_q_heads + a.cache.n_kv_heads;
        float x[8];
        unpack_bf16x8(__builtin_nontemporal_load(src + i), x);
        const uint16_t* const weight = is_q ? a.wq : is_k ? a.wk : nullptr;
        if (weight != nullptr) {
            float w[8], sum = 0.f;
            unpack_bf16x8(reinterpret_cast<const u32x4*>(weight)[part], w);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
            const float inv = 1.0f / sqrtf(row_sum<LANES>(sum) / (float)D + a.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * inv * w[j];
        }
        if (a.log2_base > 0.0 && (is_q || is_k)) {
            const float2* const cs = turn[is_k && k_pos != pos ? 1 : 0] + 4 * part;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float c = cs[j].x, s = cs[j].y, x0 = x[2 * j], x1 = x[2 * j + 1];
                x[2 * j] = x0 * c - x1 * s;
                x[2 * j + 1] = x0 * s + x1 * c;
            }
        }
        u32x4 o;
        if (is_q || !E4M3) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const bf16x2_t pair = {(__bf16)x[2 * j], (__bf16)x[2 * j + 1]};  // v_cvt_pk_bf16_f32, nearest even
                o[j] = __builtin_bit_cast(uint32_t, pair);
            }
        }
        if (is_q) {
            const size_t row = a.positions != nullptr ? (size_t)token * a.n_q_heads + head : (size_t)head * a.n_tokens + token;
            reinterpret_cast<u32x4*>(a.q_out)[row * LANES + part] = o;
            continue;
        }
        const int h = head - a.n_q_heads - (is_k ? 0 : a.cache.n_kv_heads);
        const int64_t row = kv8_row(a.cache, b, h, t);
        if (row < 0) continue;  // unmapped page: nothing to write
        uint8_t* const to = is_k ? a.cache.k : a.cache.v;
        if constexpr (E4M3) {
            uint32_t byte;
            const u32x2 codes = kv8_quantise<LANES>(x, &byte);
            reinterpret_cast<u32x2*>(to + row * D)[part] = codes;
            if (part == 0) (is_k ? a.cache.k_scale : a.cache.v_scale)[row] = (uint8_t)byte;
        } else {
            reinterpret_cast<u32x4*>(to)[row * LANES + part] = o;
        }
    }
}

}  // namespace

hipError_t launch_qk_norm_rope(int head_dim, const HeadsArgs& a, const Launch& l) {
    if (a.n_tokens < 1) return hipSuccess;
    const dim3 grid(a.n_tokens), block(kHeadsThreads);
    const bool e4m3 = a.cache.k_scale != nullptr;
    if (head_dim == 128)
        return e4m3 ? launch_kernel(qk_norm_rope_kernel<128, true>, grid, block, l, a)
                    : launch_kernel(qk_norm_rope_kernel<128, false>, grid, block, l, a);
    if (head_dim == 64)
        return e4m3 ? launch_kernel(qk_norm_rope_kernel<64, true>, grid, block, l, a)
                    : launch_kernel(qk_norm_rope_kernel<64, false>, grid, block, l, a);
    return hipErrorInvalidValue;
}

}  // namespace lara
