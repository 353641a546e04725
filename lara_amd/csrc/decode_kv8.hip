// Split-KV GQA decode over the E4M3 cache (kv8_device.h has the rows' format), gfx950.
//
// With K and V rows of codes c, c' and scales 2^a, 2^b, for one query row:
//   s_k = scale * 2^a_k * sum_d q[d] c_k[d]      p_k = exp(s_k - m)
//   O   = sum_k (p_k 2^b_k) c'_k,  l = sum_k p_k,  out = bf16(O / l)
// An E4M3 value is exact in bf16, so the products run on the bf16 matrix cores with Q unrounded; K's scale comes with the
// conversion (v_cvt_scalef32_pk_bf16_fp8), V's multiplies p (by a power of two: exact) before p is rounded to bf16, the
// one rounding of the operands (half a step, 2^-9 of p).  Sums, maxima and O are fp32.
//
// A work-group of NW waves owns a contiguous split of keys of one (sequence, kv head) for all heads of the group, so the
// cache is read once; wave w takes the split's 32-key rounds w, w + NW, ..., the next one's rows in flight behind the
// products.  There is no LDS in the loop, where the bf16 kernel passes K and V through it:
//   S^T [16 keys x 16 heads] = K . Q^T, two tiles a round.  Lane (m, g) = (l % 16, l / 16) loads the 16-byte chunks
//     g, g + 4 of key m's row, which are operand A as they lie: the order of the dims inside the sum is free, so half of
//     a chunk is the 8 values that lane gives one v_mfma_f32_16x16x32_bf16, and Q is loaded in the same order.
//   The result leaves lane (m, g) the scores of keys 4g .. 4g + 3 of both tiles for head m: the softmax is per lane, and
//     the 8 p are operand B of the second product, slots u = 0 .. 7 for keys 16 (u / 4) + 4g + u % 4.
//   O^T [D x 16 heads] += V^T . P^T.  Lane (m, g) loads D / 16 codes (dims D/16 * m ..) of the same 8 keys, a whole row by
//     16 lanes; byte t of them belongs to row m of tile t, dim D/16 * m + t.  v_perm_b32 pairs the bytes of two keys, the
//     conversion makes them a word of operand A.
// A row of length 0 writes zeros and -inf.  Rows past a split's end are cleared (a stale code may be NaN, and 0 * NaN is
// NaN) and their scores masked.
//
// The row appended by the launch: every split that holds it quantises it for itself into LDS (split 0 also writes it to
// the cache) and puts it into the registers of the round that it belongs to, so no work-group waits for another.
//
// Splits meet as in the bf16 kernel: in the launch (the last split of a (sequence, kv head) to arrive), or in a second
// launch, in the same order of sums.
#include "decode_common.h"
#include "kv8_device.h"

#include <math.h>

namespace lara {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kRoundKeys = kKv8RoundKeys;
constexpr int kMergeParts = 4;   // a head's splits are summed as s % 4 apart, then these four in order
constexpr int kMergeBatch8 = 8;  // partials in flight of one part

__device__ __forceinline__ f32x4 mfma_bf16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

// Two codes (the low or high half of `codes`) times 2^k, as a word of bf16.
template <bool HIGH>
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

template <bool CACHED, typename T>
__device__ __forceinline__ T load_stream(const void* p) {
    if constexpr (CACHED) return *reinterpret_cast<const T*>(p);
    else return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
}

// Sums part `part` (splits part, part + 4, ...) of head row `row0` (split 0's partial row; `stride` rows per split)
// against the maximum M of all of them: lane l has dims l * D / 64 ..
template <int D>
__device__ __forceinline__ void merge_part(const DecodeArgs& a, size_t row0, int stride, int n_splits, int part, float* M_out,
                                           float* L_out, float (&O)[D / 64]) {
    const int lane = threadIdx.x & 63;
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row0;
    float M = -INFINITY;
    for (int s = lane; s < n_splits; s += 64) M = fmaxf(M, ml[(size_t)s * stride].x);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    float L = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) O[i] = 0.f;
    typedef float vec __attribute__((ext_vector_type(D / 64)));
    for (int s0 = part; s0 < n_splits; s0 += kMergeParts * kMergeBatch8) {
        vec o[kMergeBatch8];
        float2 w[kMergeBatch8];
#pragma unroll
        for (int j = 0; j < kMergeBatch8; ++j) {
            const int s = s0 + j * kMergeParts;
            w[j] = make_float2(-INFINITY, 0.f);
            o[j] = vec(0.f);
            if (s < n_splits) {
                const size_t row = row0 + (size_t)s * stride;
                w[j] = reinterpret_cast<const float2*>(a.part_ml)[row];
                o[j] = reinterpret_cast<const vec*>(a.part_o + row * D)[lane];
            }
        }
#pragma unroll
        for (int j = 0; j < kMergeBatch8; ++j) {
            const float f = M == -INFINITY ? 0.f : fast_exp2(w[j].x - M);  // 0 for a split without valid keys
            L = fmaf(f, w[j].y, L);
#pragma unroll
            for (int i = 0; i < D / 64; ++i) O[i] = fmaf(f, o[j][i], O[i]);
        }
    }
    *M_out = M;
    *L_out = L;
}

// Output row (b, h, g) from the four parts of its heads in LDS ([heads][4] rows of D, and (M, L)).
template <int D>
__device__ __forceinline__ void merge_write(const DecodeArgs& a, int b, int h, int g0, int heads, const float* lds_o,
                                            const float2* lds_ml, int threads) {
    const int H_q = a.n_kv_heads * a.group;
    for (int idx = threadIdx.x; idx < heads * D; idx += threads) {
        const int g = idx / D, d = idx - g * D;
        float O = 0.f, L = 0.f;
#pragma unroll
        for (int p = 0; p < kMergeParts; ++p) {
            O += lds_o[(g * kMergeParts + p) * D + d];
            L += lds_ml[g * kMergeParts + p].y;
        }
        const size_t row = (size_t)b * H_q + h * a.group + g0 + g;
        a.out[row * D + d] = f32_to_bf16_rne(L > 0.f ? O / L : 0.f);
        if (d == 0 && a.lse != nullptr)
            a.lse[row] = L > 0.f ? (lds_ml[g * kMergeParts].x + log2f(L)) * kLn2 : -INFINITY;
    }
}

// The rows of one round in a wave's registers: K chunks, V codes, K's scale bytes (one per tile), V's (four a word).
template <int D>
struct Round {
    typedef uint32_t vword __attribute__((ext_vector_type(D / 64)));
    u32x4 k[2][D / 64];
    vword v[8];
    uint32_t ks[2], vs[2];
};

template <int D, int NW, bool PAGED, bool CACHED>
__global__ __launch_bounds__(NW * 64) void decode_kv8_kernel(DecodeArgs a) {
    constexpr int CH = D / 64;   // 16-byte chunks of a K row per lane; words of V codes per lane and key
    constexpr int VB = D / 16;   // V codes per lane and key, O tiles
    constexpr int LANES = D / 8;  // lanes that quantise a row
    typedef typename Round<D>::vword vword;

    const int split = blockIdx.x, G = a.group;
    int row = blockIdx.y;
    const bool ranked = a.longest_first && batch_is_ragged(a);
    if (a.ticket != nullptr && ranked) {  // (as in the bf16 kernel: rows in longest-first order, as work-groups start)
        __shared__ int s_row;
        if (threadIdx.x == 0) {
            const unsigned rows = gridDim.y;
            const unsigned t = (unsigned)__hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (t % rows == rows - 1) __hip_atomic_store(a.ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_row = (int)(t % rows);
        }
        __syncthreads();
        row = s_row;
    }
    const int h = row % a.n_kv_heads;
    int b = row / a.n_kv_heads;
    if (ranked) b = rank_to_sequence(a, b);
    const int unit = b * a.n_kv_heads + h, H_q = a.n_kv_heads * G;
    const int L = clamp_len(a.lens[b], a.l_max);
    const int n_splits = decode_split_count(L, a.chunk);
    if (split >= n_splits) return;  // uniform across the work-group
    const int k_begin = split * a.chunk;
    const int k_end = split == n_splits - 1 ? L : k_begin + a.chunk;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m16 = lane & 15, grp = lane >> 4;
    const int64_t row0 = (int64_t)unit * a.l_cap;
    const int32_t* const trow = PAGED ? a.block_table + (size_t)b * a.max_pages : nullptr;
    const uint8_t* const kc = reinterpret_cast<const uint8_t*>(a.kc);
    const uint8_t* const vc = reinterpret_cast<const uint8_t*>(a.vc);
    const uint8_t* const zero = reinterpret_cast<const uint8_t*>(a.zero_row);

    const int pos = a.k_new != nullptr ? a.positions[b] : -1;
    const bool has_new = pos >= 0 && pos < a.l_max;

    // Paged: 64 consecutive block-table entries, one per lane, from page pc_first on.
    int pc_first = -(1 << 30), pc_val = -1;
    auto page_of = [&](int page_idx) -> int {
        if (page_idx - pc_first >= 64 || page_idx < pc_first) {
            pc_first = page_idx;
            const int i = page_idx + lane;
            pc_val = i < a.max_pages ? trow[i] : -1;
        }
        return __builtin_amdgcn_readlane(pc_val, page_idx - pc_first);
    };
    // Rounds start at multiples of 32 and a row's region (a page) has a multiple of 64 rows, so all 32 rows of a round
    // lie inside it.
    auto load_round = [&](int key0, Round<D>& r) __attribute__((always_inline)) {
        int64_t first = row0 + key0;
        bool mapped = true;
        if constexpr (PAGED) {
            const int k0 = __builtin_amdgcn_readfirstlane(key0);
            const int page = page_of(k0 >> a.page_shift);
            mapped = page >= 0;
            first = (((int64_t)(mapped ? page : 0) * a.n_kv_heads + h) << a.page_shift) + (k0 & ((1 << a.page_shift) - 1));
        }
        const uint8_t* const k = mapped ? kc + first * D : zero;
        const uint8_t* const v = mapped ? vc + first * D : zero;
        const uint8_t* const ks = mapped ? a.k_scale + first : zero;
        const uint8_t* const vs = mapped ? a.v_scale + first : zero;
        const int step = mapped ? D : 0, one = mapped ? 1 : 0;  // (an unmapped page: every row is the zero row)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int j = 0; j < CH; ++j)
                r.k[t][j] = load_stream<CACHED, u32x4>(k + (16 * t + m16) * step + 16 * (grp + 4 * j));
            r.ks[t] = ks[(16 * t + m16) * one];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            r.v[u] = load_stream<CACHED, vword>(v + (16 * (u >> 2) + 4 * grp + (u & 3)) * step + VB * m16);
#pragma unroll
        for (int t = 0; t < 2; ++t) r.vs[t] = *reinterpret_cast<const uint32_t*>(vs + (16 * t + 4 * grp) * one);
    };

    const int n_rounds = (k_end - k_begin + kRoundKeys - 1) / kRoundKeys;
    Round<D> next;
    int r = wave;
    if (r < n_rounds) load_round(k_begin + r * kRoundKeys, next);

    // The appended row: wave 0 quantises K's, wave 1 V's.
    __shared__ __attribute__((aligned(16))) uint8_t new_codes[2][D];
    __shared__ uint8_t new_scale[2];
    const bool new_here = has_new && (split == 0 || (pos >= k_begin && pos < k_end));
    if (new_here) {
        if (wave < 2 && lane < LANES) {
            float x[8];
            unpack_bf16x8(reinterpret_cast<const u32x4*>((wave ? a.v_new : a.k_new) + (size_t)unit * D)[lane], x);
            uint32_t byte;
            const u32x2 c = kv8_quantise<LANES>(x, &byte);
            reinterpret_cast<u32x2*>(new_codes[wave])[lane] = c;
            if (lane == 0) new_scale[wave] = (uint8_t)byte;
            if (split == 0) {
                const int64_t at = PAGED ? paged_row(trow, a.page_shift, a.n_kv_heads, h, pos) : row0 + pos;
                if (at >= 0) {  // (unmapped: not written)
                    reinterpret_cast<u32x2*>(const_cast<uint8_t*>(wave ? vc : kc) + at * D)[lane] = c;
                    if (lane == 0) (wave ? a.v_scale : a.k_scale)[at] = (uint8_t)byte;
                }
            }
        }
        __syncthreads();
    }

    // Q^T operand: lane (m, g) holds, for chunk j's half i, dims 16 (g + 4j) + 8i .. of head m (heads past G are zero).
    u32x4 qb[2 * CH];
    {
        const u32x4* qp = reinterpret_cast<const u32x4*>(a.q + ((size_t)b * H_q + h * G + (m16 < G ? m16 : 0)) * D);
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) qb[2 * j + i] = m16 < G ? qp[2 * (grp + 4 * j) + i] : u32x4{0u, 0u, 0u, 0u};
    }
    f32x4 o_acc[VB];  // tile t: dims VB * (4g + i) + t of head m in register i
#pragma unroll
    for (int t = 0; t < VB; ++t) o_acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_lane = 0.f;

    for (; r < n_rounds; r += NW) {
        const int key0 = k_begin + r * kRoundKeys;
        Round<D> cur = next;
        if (r + NW < n_rounds) load_round(key0 + NW * kRoundKeys, next);
        if (key0 + kRoundKeys > k_end || (has_new && pos >= key0 && pos < key0 + kRoundKeys)) {
            const int at = has_new ? pos - key0 : -1;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const bool fresh = at == 16 * t + m16 && key0 + at < k_end;
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const u32x4 w = reinterpret_cast<const u32x4*>(new_codes[0])[grp + 4 * j];
                    cur.k[t][j] = fresh ? w : cur.k[t][j];
                }
                if (fresh) cur.ks[t] = new_scale[0];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int key = 16 * (u >> 2) + 4 * grp + (u & 3);
                const vword w = reinterpret_cast<const vword*>(new_codes[1])[m16];
                const bool past = key0 + key >= k_end;
                cur.v[u] = past ? vword(0u) : key == at ? w : cur.v[u];
                if (key == at && !past) {
                    const uint32_t shift = 8 * (u & 3);
                    cur.vs[u >> 2] = (cur.vs[u >> 2] & ~(0xFFu << shift)) | ((uint32_t)new_scale[1] << shift);
                }
            }
        }

        // S^T, two tiles of 16 keys.
        float s[8];
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float scale = kv8_scale(cur.ks[t]);
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < CH; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t lo = cur.k[t][j][2 * i], hi = cur.k[t][j][2 * i + 1];
                    const u32x4 ka = {codes_to_bf16<false>(lo, scale), codes_to_bf16<true>(lo, scale),
                                      codes_to_bf16<false>(hi, scale), codes_to_bf16<true>(hi, scale)};
                    acc = mfma_bf16(ka, qb[2 * j + i], acc);
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[4 * t + i] = key0 + 16 * t + 4 * grp + i < k_end ? acc[i] * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, s[4 * t + i]);
            }
        }
        mx = pair_max32(pair_max16(mx));
        const float m_cand = fmaxf(m_run, mx);
        if (__ballot(m_cand > m_run + kRescaleSlack) != 0) {
            const float corr = m_cand == -INFINITY ? 1.f : fast_exp2(m_run - m_cand);
            m_run = m_cand;
            l_lane *= corr;
#pragma unroll
            for (int t = 0; t < VB; ++t) o_acc[t] *= corr;
        }
        float p[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            p[u] = s[u] == -INFINITY ? 0.f : fast_exp2(s[u] - m_run);
            l_lane += p[u];
            p[u] *= kv8_scale((cur.vs[u >> 2] >> (8 * (u & 3))) & 0xFFu);
        }
        const u32x4 pb = {pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};

        // O^T += V^T . P^T, four tiles per word of codes.
#pragma unroll
        for (int w = 0; w < CH; ++w) {
            u32x4 va[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = __builtin_amdgcn_perm(cur.v[2 * i + 1][w], cur.v[2 * i][w], 0x05010400u);
                const uint32_t hi = __builtin_amdgcn_perm(cur.v[2 * i + 1][w], cur.v[2 * i][w], 0x07030602u);
                va[0][i] = codes_to_bf16<false>(lo, 1.f);
                va[1][i] = codes_to_bf16<true>(lo, 1.f);
                va[2][i] = codes_to_bf16<false>(hi, 1.f);
                va[3][i] = codes_to_bf16<true>(hi, 1.f);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) o_acc[4 * w + c] = mfma_bf16(va[c], pb, o_acc[4 * w + c]);
        }
    }

    // ---- the waves of this work-group: [NW][G] rows of D (+ 4: bank conflicts), then (m, l)
    constexpr int OS = D + 4;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float* const lds_o = lds;
    float2* const lds_ml = reinterpret_cast<float2*>(lds + NW * G * OS);
    {
        const float l_head = pair_sum32(pair_sum16(l_lane));
        if (m16 < G) {
            float* const to = lds_o + (wave * G + m16) * OS;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < VB; t += 4)
                    *reinterpret_cast<f32x4*>(to + VB * (4 * grp + i) + t) =
                        f32x4{o_acc[t][i], o_acc[t + 1][i], o_acc[t + 2][i], o_acc[t + 3][i]};
            if (grp == 0) lds_ml[wave * G + m16] = make_float2(m_run, l_head);
        }
    }
    __syncthreads();
    const bool single = n_splits == 1, fused = !single && a.arrivals != nullptr;
    for (int idx = threadIdx.x; idx < G * D; idx += NW * 64) {
        const int g = idx / D, d = idx - g * D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, lds_ml[w * G + g].x);
        float O = 0.f, Ls = 0.f;
        if (M != -INFINITY) {
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float2 ml = lds_ml[w * G + g];
                const float f = fast_exp2(ml.x - M);  // 0 for a wave without rounds
                O = fmaf(f, lds_o[(w * G + g) * OS + d], O);
                Ls = fmaf(f, ml.y, Ls);
            }
        }
        if (single) {
            const size_t to = (size_t)b * H_q + h * G + g;
            a.out[to * D + d] = f32_to_bf16_rne(Ls > 0.f ? O / Ls : 0.f);
            if (d == 0 && a.lse != nullptr) a.lse[to] = Ls > 0.f ? (M + log2f(Ls)) * kLn2 : -INFINITY;
        } else {
            const size_t to = ((size_t)unit * a.max_splits + split) * G + g;
            if (fused) {  // agent-scope stores: seen across the XCDs without an L2 write-back
                __hip_atomic_store(&a.part_o[to * D + d], O, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (d == 0) {
                    __hip_atomic_store(&a.part_ml[to * 2], M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    __hip_atomic_store(&a.part_ml[to * 2 + 1], Ls, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            } else {
                a.part_o[to * D + d] = O;
                if (d == 0) reinterpret_cast<float2*>(a.part_ml)[to] = make_float2(M, Ls);
            }
        }
    }
    if (!fused) return;
    // The last split of the (sequence, kv head) to arrive merges them: its threads' partials are stored before thread 0's
    // release increment, the increment that reads n_splits - 1 acquires the others', and resets the counter.
    __shared__ int is_last;
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    __syncthreads();
    if (threadIdx.x == 0) {
        const int prev = __hip_atomic_fetch_add(&a.arrivals[unit], 1, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT);
        is_last = prev == n_splits - 1;
        if (is_last) {
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
            __hip_atomic_store(&a.arrivals[unit], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    __syncthreads();
    if (!is_last) return;
    static_assert(NW >= kMergeParts, "the merge's LDS is inside the waves'");
    float2* const merge_ml = reinterpret_cast<float2*>(lds + kMergeParts * G * D);
    for (int task = wave; task < G * kMergeParts; task += NW) {
        const int g = task / kMergeParts, part = task - g * kMergeParts;
        float M, Ls, O[D / 64];
        merge_part<D>(a, (size_t)unit * a.max_splits * G + g, G, n_splits, part, &M, &Ls, O);
#pragma unroll
        for (int i = 0; i < D / 64; ++i) lds[task * D + lane * (D / 64) + i] = O[i];
        if (lane == 0) merge_ml[task] = make_float2(M, Ls);
    }
    __syncthreads();
    merge_write<D>(a, b, h, 0, G, lds, merge_ml, NW * 64);
}

// The merge launch: a work-group per (sequence, kv head, head of the group), a wave per part.
template <int D>
__global__ __launch_bounds__(kMergeParts * 64) void decode_kv8_merge_kernel(DecodeArgs a) {
    const int unit = blockIdx.x / a.group, g = blockIdx.x - unit * a.group;
    const int b = unit / a.n_kv_heads, h = unit - b * a.n_kv_heads;
    const int n_splits = decode_split_count(clamp_len(a.lens[b], a.l_max), a.chunk);
    if (n_splits <= 1) return;  // written by the split kernel
    __shared__ float lds_o[kMergeParts * D];
    __shared__ float2 lds_ml[kMergeParts];
    const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
    float M, Ls, O[D / 64];
    merge_part<D>(a, (size_t)unit * a.max_splits * a.group + g, a.group, n_splits, part, &M, &Ls, O);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) lds_o[part * D + lane * (D / 64) + i] = O[i];
    if (lane == 0) lds_ml[part] = make_float2(M, Ls);
    __syncthreads();
    merge_write<D>(a, b, h, g, 1, lds_o, lds_ml, kMergeParts * 64);
}

template <int D, int NW>
hipError_t launch_kv8_t(const DecodeArgs& a, const Launch& l) {
    const dim3 grid(a.max_splits, a.batch * a.n_kv_heads), block(NW * 64);
    const size_t lds = ((size_t)NW * a.group * (D + 4) + NW * a.group * 2) * sizeof(float);
    void (*const kernel)(DecodeArgs) =
        a.block_table != nullptr ? (a.cached ? decode_kv8_kernel<D, NW, true, true> : decode_kv8_kernel<D, NW, true, false>)
                                 : (a.cached ? decode_kv8_kernel<D, NW, false, true> : decode_kv8_kernel<D, NW, false, false>);
    return launch_kernel_lds(kernel, grid, block, lds, l, a);
}

}  // namespace

bool decode_kv8_supported(int head_dim, int group) { return (head_dim == 64 || head_dim == 128) && group >= 1 && group <= 16; }

hipError_t launch_decode_kv8(int head_dim, const DecodeArgs& a, const Launch& l) {
    if (!decode_kv8_supported(head_dim, a.group)) return hipErrorInvalidValue;
    if (a.waves == kDecodeWavesSmall)
        return head_dim == 128 ? launch_kv8_t<128, kDecodeWavesSmall>(a, l) : launch_kv8_t<64, kDecodeWavesSmall>(a, l);
    if (a.waves == kDecodeWaves)
        return head_dim == 128 ? launch_kv8_t<128, kDecodeWaves>(a, l) : launch_kv8_t<64, kDecodeWaves>(a, l);
    return hipErrorInvalidValue;
}

hipError_t launch_decode_kv8_merge(int head_dim, const DecodeArgs& a, const Launch& l) {
    const dim3 grid(a.batch * a.n_kv_heads * a.group), block(kMergeParts * 64);
    if (head_dim == 128) return launch_kernel(decode_kv8_merge_kernel<128>, grid, block, l, a);
    if (head_dim == 64) return launch_kernel(decode_kv8_merge_kernel<64>, grid, block, l, a);
    return hipErrorInvalidValue;
}

}  // namespace lara
