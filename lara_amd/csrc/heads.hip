// Norms of the query and key heads with the position rotation, into Q and the cache, in one pass.
//
// Per head row h of D values (fp32 from bf16):  y = h / sqrt(mean(h^2) + eps) * w  (w nullptr: no norm), then each pair
// (2p, 2p + 1) of y is turned by position * base^(-2p / D); V rows go as they are.  Everything is fp32 up to one rounding
// at the end: to bf16, or to a row of the E4M3 cache.  The angle and its sine and cosine are 64-bit (an fp32 angle is off
// by 2^-25 of itself: 0.03 rad at position 10^6).
//
// D / 8 lanes hold a head row, so its sum of squares (and an E4M3 row's maximum) is three or four lane exchanges, and a
// lane's four pairs are the same in every head that it takes.  A work-group is a token (two of a prompt at D 64, as many
// rows), so an angle is made once for all of its heads; three rows a thread are on their way at once, the first ones and
// the weights while the angles are computed.
//
// Bound by memory for long prompts: 8192 tokens of 32 + 16 heads of 128 (185 MB) in 28.3 us beside other launches, 6.5 TB/s
// (32 alone; a load and a weight at a time 37); 2048 (50 MB) 9.3 / 12.2, one wave of work-groups whose vector
// instructions and loads take turns; 4000 of 48 heads of 64 11.5 alone, 13.4 with a token a work-group.  Two tokens a
// work-group at D 128: 14.2 at 2048, 36 at 8192.  Registers for 8 work-groups a CU matter: with 80 (weights and angles kept
// as fp32) 2048 take 14.6.  A step of 64 sequences (1.4 MB) is a launch: 4.5 alone, 5.1 without the loads ahead.
//
// The other forms turn the first rotary_dim dims only, as pairs (2p, 2p + 1) or halves (p, p + rotary_dim / 2), by angles per
// position that the host computed in 64 bits (turns, so that whole ones go before the angle is rounded and sine and cosine
// can be fp32), and multiply both by a magnitude.  They cost what the plain form does: 2048 tokens as above 9.7 / 12.2, a
// step of 64 sequences into the E4M3 cache 4.2 / 4.8.
#include "kv8_device.h"

#include <math.h>

#include <type_traits>

namespace lara {
namespace {

constexpr int kHeadsThreads = 256;
constexpr int kHeadsBatch = 3;

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

// How a row turns: whole, pairs side by side, base^(-2p / D) (HeadsArgs); or as RotaryArgs say.
enum Form { kPlain, kPairs, kHalves };
template <Form FORM>
using FormArgs = std::conditional_t<FORM == kPlain, HeadsArgs, RotaryArgs>;

// TOKENS tokens a work-group (one of the step form); a thread keeps its token and its place in a row.
template <int D, bool E4M3, int TOKENS, Form FORM>
__global__ __launch_bounds__(kHeadsThreads) void qk_norm_rope_kernel(FormArgs<FORM> a) {
    constexpr int LANES = D / 8, PAIRS = D / 2;
    const int token0 = wide_block() * TOKENS;
    if (token0 >= a.n_tokens) return;  // (the whole work-group)
    const int tokens = TOKENS == 1 || a.n_tokens - token0 >= TOKENS ? TOKENS : a.n_tokens - token0;
    const int part = threadIdx.x % LANES;
    int b = a.b, pos0 = a.pos_base + token0, k_pos0 = a.k_pos_base + token0, t0 = a.row0 + token0;
    if (TOKENS == 1 && a.positions != nullptr) {  // one token of each sequence
        b = token0;
        pos0 = k_pos0 = a.positions[token0];
        t0 = a.rows != nullptr ? a.rows[token0] : pos0;
        if (pos0 < 0 || t0 < 0 || t0 >= a.cache.l_max) return;  // (the whole work-group) nothing of this sequence is written
    }
    const int heads = a.n_q_heads + 2 * a.cache.n_kv_heads, chunks = heads * TOKENS * LANES;
    // A lane's 8 values are two runs of 4 dims, one behind the other; where halves turn, the lanes of the dims that turn have
    // a run of each half, so that both values of a pair are in one lane in every form.
    int run0 = 8 * part, run1 = 8 * part + 4;
    bool turning = true;
    if constexpr (FORM != kPlain) turning = 8 * part < a.rotary_dim;
    if constexpr (FORM == kHalves)
        if (turning) run0 = 4 * part, run1 = a.rotary_dim / 2 + 4 * part;
    auto load_runs = [&](const uint16_t* row) __attribute__((always_inline)) {
        const u32x2 lo = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(row + run0));
        const u32x2 hi = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(row + run1));
        return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    auto store_runs = [&](uint16_t* row, const u32x4& w) __attribute__((always_inline)) {
        *reinterpret_cast<u32x2*>(row + run0) = u32x2{w[0], w[1]};
        *reinterpret_cast<u32x2*>(row + run1) = u32x2{w[2], w[3]};
    };
    // A batch of values is loaded at once, the first ahead of the angles.
    u32x4 in[kHeadsBatch];
    auto load = [&](int from) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < kHeadsBatch; ++k) {
            const int i = from + k * kHeadsThreads, of = i / LANES % TOKENS;
            if (i >= chunks || of >= tokens) continue;
            const uint16_t* const row = a.x + (size_t)(token0 + of) * a.ld;
            if constexpr (FORM == kHalves)
                in[k] = load_runs(row + i / (LANES * TOKENS) * D);
            else
                in[k] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(row) + i / (LANES * TOKENS) * LANES + part);
        }
    };
    load(threadIdx.x);
    u32x4 wq = {}, wk = {};
    if constexpr (FORM == kHalves) {
        if (a.wq != nullptr) wq = load_runs(a.wq);
        if (a.wk != nullptr) wk = load_runs(a.wk);
    } else {
        if (a.wq != nullptr) wq = reinterpret_cast<const u32x4*>(a.wq)[part];
        if (a.wk != nullptr) wk = reinterpret_cast<const u32x4*>(a.wk)[part];
    }
    __shared__ float2 turn[2][TOKENS][PAIRS];
    if constexpr (FORM != kPlain) {
        const int sets = k_pos0 != pos0 ? 2 : 1;
        for (int i = threadIdx.x; i < sets * TOKENS * PAIRS; i += kHeadsThreads) {
            const int p = i % PAIRS, of = i / PAIRS % TOKENS, set = i / (PAIRS * TOKENS);
            if (2 * p >= a.rotary_dim) continue;
            // The angle in turns: its whole ones go, in 64 bits, before it is rounded (to 2^-25 of at most half a turn).
            const double t = (double)((set ? k_pos0 : pos0) + of) * a.turns[p];
            float s, c;
            sincospif(2.f * (float)(t - rint(t)), &s, &c);
            turn[set][of][p] = make_float2(c * a.magnitude, s * a.magnitude);
        }
        __syncthreads();
    } else if (a.log2_base > 0.0) {
        const int sets = k_pos0 != pos0 ? 2 : 1;
        for (int i = threadIdx.x; i < sets * TOKENS * PAIRS; i += kHeadsThreads) {
            const int p = i % PAIRS, of = i / PAIRS % TOKENS, set = i / (PAIRS * TOKENS);
            double sd, cd;
            sincos((double)((set ? k_pos0 : pos0) + of) * exp2(-2.0 * p / D * a.log2_base), &sd, &cd);
            turn[set][of][p] = make_float2((float)cd, (float)sd);
        }
        __syncthreads();
    }
    auto process = [&](int i, const u32x4& words) __attribute__((always_inline)) {  // (a row's lanes stay together)
        const int of = i / LANES % TOKENS, token = token0 + of;
        if (i >= chunks || of >= tokens) return;
        const int head = i / (LANES * TOKENS);
        const bool is_q = head < a.n_q_heads, is_k = !is_q && head < a.n_q_heads + a.cache.n_kv_heads;
        float x[8];
        unpack_bf16x8(words, x);
        if (is_q ? a.wq != nullptr : is_k && a.wk != nullptr) {
            float w[8], sum = 0.f;
            unpack_bf16x8(is_q ? wq : wk, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = fmaf(x[j], x[j], sum);
            const float inv = rsqrtf(row_sum<LANES>(sum) * (1.0f / D) + a.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = x[j] * inv * w[j];
        }
        bool turns = turning;
        if constexpr (FORM == kPlain) turns = a.log2_base > 0.0;
        if (turns && (is_q || is_k)) {
            const float2* const cs = turn[is_k && k_pos0 != pos0 ? 1 : 0][of] + 4 * part;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                constexpr int STEP = FORM == kHalves ? 1 : 2, FAR = FORM == kHalves ? 4 : 1;
                const float c = cs[j].x, s = cs[j].y, x0 = x[STEP * j], x1 = x[STEP * j + FAR];
                x[STEP * j] = x0 * c - x1 * s;
                x[STEP * j + FAR] = x0 * s + x1 * c;
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
            if constexpr (FORM == kHalves)
                store_runs(a.q_out + row * D, o);
            else
                reinterpret_cast<u32x4*>(a.q_out)[row * LANES + part] = o;
            return;
        }
        const int h = head - a.n_q_heads - (is_k ? 0 : a.cache.n_kv_heads);
        const int64_t row = kv8_row(a.cache, b, h, t0 + of);
        if (row < 0) return;  // unmapped page: nothing to write
        uint8_t* const to = is_k ? a.cache.k : a.cache.v;
        if constexpr (E4M3) {
            uint32_t byte;
            const u32x2 codes = kv8_quantise<LANES>(x, &byte);
            if constexpr (FORM == kHalves) {
                *reinterpret_cast<uint32_t*>(to + row * D + run0) = codes[0];
                *reinterpret_cast<uint32_t*>(to + row * D + run1) = codes[1];
            } else {
                reinterpret_cast<u32x2*>(to + row * D)[part] = codes;
            }
            if (part == 0) (is_k ? a.cache.k_scale : a.cache.v_scale)[row] = (uint8_t)byte;
        } else if constexpr (FORM == kHalves) {
            store_runs(reinterpret_cast<uint16_t*>(to) + row * D, o);
        } else {
            reinterpret_cast<u32x4*>(to)[row * LANES + part] = o;
        }
    };
    for (int i = threadIdx.x; i < chunks; i += kHeadsBatch * kHeadsThreads) {
#pragma unroll
        for (int k = 0; k < kHeadsBatch; ++k) process(i + k * kHeadsThreads, in[k]);
        load(i + kHeadsBatch * kHeadsThreads);
    }
}

}  // namespace

template <int D, int TOKENS, Form FORM>
static hipError_t launch_tokens(const FormArgs<FORM>& a, const Launch& l) {
    const dim3 grid = wide_grid((a.n_tokens + TOKENS - 1) / TOKENS), block(kHeadsThreads);
    return a.cache.k_scale != nullptr ? launch_kernel(qk_norm_rope_kernel<D, true, TOKENS, FORM>, grid, block, l, a)
                                      : launch_kernel(qk_norm_rope_kernel<D, false, TOKENS, FORM>, grid, block, l, a);
}

template <Form FORM>
static hipError_t launch_form(int head_dim, const FormArgs<FORM>& a, const Launch& l) {
    if (a.n_tokens < 1) return hipSuccess;
    if (head_dim == 128) return launch_tokens<128, 1, FORM>(a, l);
    if (head_dim == 64) return a.positions == nullptr ? launch_tokens<64, 2, FORM>(a, l) : launch_tokens<64, 1, FORM>(a, l);
    return hipErrorInvalidValue;
}

hipError_t launch_qk_norm_rope(int head_dim, const HeadsArgs& a, const Launch& l) { return launch_form<kPlain>(head_dim, a, l); }

hipError_t launch_qk_norm_rotary(int head_dim, const RotaryArgs& a, const Launch& l) {
    return a.halves ? launch_form<kHalves>(head_dim, a, l) : launch_form<kPairs>(head_dim, a, l);
}

}  // namespace lara
