// What the decode kernels over bf16 and E4M3 caches share: the softmax's small helpers and the order in which a
// launch takes the batch's sequences.
#pragma once

#include "gqa_internal.h"

#include <limits.h>
#include <math.h>

namespace lara {
namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

constexpr float kLn2 = 0.693147180559945309f;

// Lazy rescaling: the running max a wave's p values are taken against moves only when a
// score exceeds it by more than this (log2 units), so p <= 2^8 and most rounds skip the
// rescale of O.  The result is the same softmax; only fp32 rounding differs.
constexpr float kRescaleSlack = 8.0f;

__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
    const bf16x2_t v = {(__bf16)lo, (__bf16)hi};  // v_cvt_pk_bf16_f32, round to nearest even
    return __builtin_bit_cast(uint32_t, v);
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Sums (m, l, O) of a softmax are joined at the largest m.  Where that is -inf, no score was above it: l and O are 0 (no
// key) or NaN (scores of NaN, which a maximum passes over), and both come through weights of 0.
__device__ __forceinline__ float softmax_base(float m) { return m == -INFINITY ? 0.f : m; }
// A row and its natural-log sum: 0 and -inf without keys (l is 1 at least where there is a score that is a number), NaN
// with a score of NaN.
__device__ __forceinline__ float softmax_out(float o, float l) { return l == 0.f ? 0.f : o / l; }
__device__ __forceinline__ float softmax_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

__device__ __forceinline__ int clamp_len(int len, int l_max) {
    return len < 0 ? 0 : (len > l_max ? l_max : len);
}

// The sequence of rank `rank` when the batch is ordered longest first.  Every wave computes it
// for itself from the lengths (no LDS, no barrier); a batch of equal lengths keeps index order.
//  * Up to 64 sequences (one per lane): exact -- by attended length, ties in index order (a wave
//    min/max, then a batch-long loop of lane reads).
//  * More: by length bucket (kBuckets equal slices of 0..l_max), longest bucket first, index
//    order inside a bucket -- a histogram of ballots over 64-sequence chunks, then the rank's
//    bucket and its position among that bucket's members.
constexpr int kBuckets = 16;

__device__ __forceinline__ int length_bucket(const DecodeArgs& a, int s) {
    const int L = clamp_len(a.lens[s], a.l_max);
    return (int)(((int64_t)L * kBuckets) / ((int64_t)a.l_max + 1));
}

// Whether the batch's attended lengths differ (every lane of the wave gets the same answer).
__device__ bool batch_is_ragged(const DecodeArgs& a) {
    const int lane = threadIdx.x & 63;
    int lo = INT_MAX, hi = -1;
    for (int s = lane; s < a.batch; s += 64) {
        const int L = clamp_len(a.lens[s], a.l_max);
        lo = L < lo ? L : lo;
        hi = L > hi ? L : hi;
    }
    return __reduce_min_sync(~0ull, lo) != __reduce_max_sync(~0ull, hi);
}

__device__ int rank_to_sequence(const DecodeArgs& a, int rank) {
    const int lane = threadIdx.x & 63;
    if (a.batch <= 64) {
        const int mine = lane < a.batch ? clamp_len(a.lens[lane], a.l_max) : -1;
        const int lo = __reduce_min_sync(~0ull, lane < a.batch ? mine : INT_MAX);
        const int hi = __reduce_max_sync(~0ull, mine);
        if (lo == hi) return rank;
        int before = 0;  // sequences ordered ahead of this lane's
        for (int j = 0; j < a.batch; ++j) {
            const int other = __builtin_amdgcn_readlane(mine, j);
            before += (other > mine) || (other == mine && j < lane);
        }
        const unsigned long long hit = __ballot(lane < a.batch && before == rank);
        return hit ? (int)__builtin_ctzll(hit) : rank;
    }
    // Bucket histogram (wave-uniform counts).
    int count[kBuckets];
#pragma unroll
    for (int k = 0; k < kBuckets; ++k) count[k] = 0;
    for (int c0 = 0; c0 < a.batch; c0 += 64) {
        const int s = c0 + lane;
        const int kb = s < a.batch ? length_bucket(a, s) : -1;
#pragma unroll
        for (int k = 0; k < kBuckets; ++k) count[k] += __popcll(__ballot(kb == k));
    }
    // The rank's bucket (longest first) and its position among the bucket's members.
    int want = -1, pos = rank;
#pragma unroll
    for (int k = kBuckets - 1; k >= 0; --k) {
        if (want < 0) {
            if (pos < count[k]) want = k;
            else pos -= count[k];
        }
    }
    if (want < 0) return rank;  // rank outside the batch: not reached for grid rows < batch
    for (int c0 = 0; c0 < a.batch; c0 += 64) {
        const int s = c0 + lane;
        const bool member = s < a.batch && length_bucket(a, s) == want;
        const unsigned long long m = __ballot(member);
        const int n = __popcll(m);
        if (pos < n) {
            // the member lane with `pos` members below it
            const int below = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
            const unsigned long long hit = __ballot(member && below == pos);
            return c0 + (int)__builtin_ctzll(hit);
        }
        pos -= n;
    }
    return rank;
}

}  // namespace
}  // namespace lara
