// Eviction from the cache: of every (sequence, kv head) with more than `keep` rows the first `sinks`, the last `recent` and
// the heaviest between stay, by the mass that they have; equal ones go by their index, NaN counts as less than anything.
// The rows that stay move together, in their order, to the first `keep`.
//
// Selection, a work-group per (sequence, kv head): masses are taken as unsigned numbers of the same order, and rows that stay
// in any case have the greatest; the least that stays is found by its bits, 11, 11 and 10 at a time, from a histogram of those
// that share the bits found so far.  A thread has a run of rows, so that the rows that stay in the runs before give its own
// their places.  It is latency: 8 us for eight sequences of 8 kv heads and 8192 rows, 15 us for 64 of them.  (Rows in turn over
// the lanes with ballots for places take 13 and 21 us: the code of a ballot per 64 rows is long, and runs once.)
//
// Moving, in place: row j comes from row kept[j] >= j, and kept rises, so a work-group that takes the rows in order, a batch
// at a time, has read all that a batch's stores may overwrite once the batch itself is read; the next batch's loads may even
// pass them.  Rows do not mix along their bytes, so a (sequence, kv head) is shared out by K and V and by columns, which
// need nothing of each other: no work-group waits for another.  Scales and masses are one more work-group's.  The memory
// bounds it: 64 sequences of 8 kv heads, 2048 rows of 256 bytes kept of 8192, 222 us (read and written at 4.9 TB/s).
#include "decode_common.h"
#include "kv8_device.h"

namespace lara {
namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kSelectHeld = 2;  // steps of four masses that a thread keeps in registers; those past them are read again
constexpr int kBins = 2048;
constexpr int kMoveThreads = 512, kMoveBatch = 8;  // 16-byte words of a batch per thread

// The order of masses as that of unsigned numbers from 2 to 2^32 - 2: NaN has 1, -0 is 0.
__device__ __forceinline__ uint32_t mass_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 1u : u >> 31 ? ~u : u | 0x80000000u;
}
constexpr uint32_t kSure = 0xFFFFFFFFu;  // a row that stays whatever its mass

// The sums of the waves' numbers before wave `wave`'s, lane by lane; `of` holds one per wave.
__device__ __forceinline__ int waves_before(const int* of, int wave, int lane) {
    const int n = lane < kSelectWaves ? of[lane] : 0;
    return __builtin_amdgcn_readlane(wave_scan(n) - n, wave);
}

__global__ __launch_bounds__(kSelectThreads, 8) void evict_select_kernel(EvictArgs a) {
    const int unit = wide_block(), b = unit / a.cache.n_kv_heads;
    if (b >= a.batch) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int L = clamp_len(a.lens[b], a.cache.l_max);
    if (unit == b * a.cache.n_kv_heads && tid == 0) a.lens_copy[b] = L;
    int32_t* const kept = a.kept + (size_t)unit * a.keep;
    if (L <= a.keep) {
        for (int j = tid; j < a.keep; j += kSelectThreads) kept[j] = j < L ? j : -1;
        return;
    }
    const float* const mass = a.mass + (size_t)unit * a.mass_ld;
    // A thread has one run of rows, four a step.
    const int lo = a.sinks, hi = L - a.recent, per = 4 * ((L + 4 * kSelectThreads - 1) / (4 * kSelectThreads)), first = tid * per;
    struct Step {
        uint32_t k[4];
    };
    auto step = [&](int t) __attribute__((always_inline)) {
        float m[4] = {0.f, 0.f, 0.f, 0.f};
        if (t + 4 <= L) {
            __builtin_memcpy(m, mass + t, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (t + i < L) m[i] = mass[t + i];
        }
        Step s;
#pragma unroll
        for (int i = 0; i < 4; ++i) s.k[i] = t + i >= L ? 0u : t + i < lo || t + i >= hi ? kSure : mass_key(m[i]);
        return s;
    };
    Step held[kSelectHeld];
#pragma unroll
    for (int c = 0; c < kSelectHeld; ++c)
        if (4 * c < per) held[c] = step(first + 4 * c);
    // Calls f(row, key) for the thread's rows in their order; rows past L have the key 0, which nothing else has.
    auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < kSelectHeld; ++c)
            if (4 * c < per)
#pragma unroll
                for (int i = 0; i < 4; ++i) f(first + 4 * c + i, held[c].k[i]);
#pragma unroll 1
        for (int c = kSelectHeld; 4 * c < per; ++c) {
            const Step s = step(first + 4 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) f(first + 4 * c + i, s.k[i]);
        }
    };
    __shared__ int hist[3][kBins];
    __shared__ int total[2][kSelectWaves];
    __shared__ int found[3][2];
    for (int i = tid; i < 3 * kBins; i += kSelectThreads) hist[0][i] = 0;
    __syncthreads();
    uint32_t least = 0, mask = 0;
    int quota = a.keep;  // rows that stay of those whose key begins with the bits of `least`: in the end, is it
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        each([&](int, uint32_t k) __attribute__((always_inline)) {
            if (k != 0 && (k & mask) == least) atomicAdd(&hist[pass][(k >> shift) & (bins - 1)], 1);
        });
        __syncthreads();
        // Bins from the top, kPer a thread; the one in which the count reaches the quota is it.
        constexpr int kPer = kBins / kSelectThreads;
        const int top = bins - 1 - kPer * tid;
        int n[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum += n[i] = top >= i ? hist[pass][top - i] : 0;
        const int upto = wave_scan(sum);
        if (lane == 63) total[pass & 1][wave] = upto;
        __syncthreads();
        int before = waves_before(total[pass & 1], wave, lane) + upto - sum;
        if (before < quota && quota <= before + sum) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                if (before < quota && quota <= before + n[i]) {
                    found[pass][0] = top - i;
                    found[pass][1] = quota - before;
                }
                before += n[i];
            }
        }
        __syncthreads();
        least |= (uint32_t)found[pass][0] << shift;
        mask |= (uint32_t)(bins - 1) << shift;
        quota = found[pass][1];
    }
    // Places: what stays of the waves, lanes and rows before.
    int more = 0, even = 0;
    each([&](int, uint32_t k) __attribute__((always_inline)) {
        more += k > least ? 1 : 0;
        even += k == least ? 1 : 0;
    });
    const int more_upto = wave_scan(more), even_upto = wave_scan(even);
    __shared__ int more_of[kSelectWaves], even_of[kSelectWaves];
    if (lane == 63) {
        more_of[wave] = more_upto;
        even_of[wave] = even_upto;
    }
    __syncthreads();
    more = waves_before(more_of, wave, lane) + more_upto - more;
    even = waves_before(even_of, wave, lane) + even_upto - even;
    each([&](int t, uint32_t k) __attribute__((always_inline)) {
        if (k > least || (k == least && even < quota)) kept[more + min(even, quota)] = t;
        more += k > least ? 1 : 0;
        even += k == least ? 1 : 0;
    });
}

// What a value held in registers needs before a barrier that stands for "read by all".
template <typename T>
__device__ __forceinline__ void arrived(T& v) {
    asm volatile("" : "+v"(v));
}

// Blocks: (sequence, kv head), then K's slices, V's slices, and the one for scales and masses.
__global__ __launch_bounds__(kMoveThreads) void evict_move_kernel(EvictArgs a) {
    const uint32_t block = wide_block();
    const int per = 2 * a.slices + 1;
    const int unit = block / per, slice = block - unit * per;
    const int b = unit / a.cache.n_kv_heads, h = unit - b * a.cache.n_kv_heads;
    if (b >= a.batch) return;
    const int L = a.lens_copy[b], keep = a.keep;
    const int32_t* const kept = a.kept + (size_t)unit * keep;
    if (slice == 2 * a.slices) {
        const float* const mass = a.mass + (size_t)unit * a.mass_ld;
        float* const new_mass = a.new_mass + (size_t)unit * a.mass_ld;
        if (h == 0 && threadIdx.x == 0) a.new_lens[b] = min(L, keep);
        if (L <= keep) {
            if (mass != new_mass)
                for (int t = threadIdx.x; t < L; t += kMoveThreads) new_mass[t] = mass[t];
            return;
        }
        for (int j0 = 0; j0 < keep; j0 += kMoveThreads * kMoveBatch) {
            float m[kMoveBatch];
            int ks[kMoveBatch], vs[kMoveBatch];
            int64_t to[kMoveBatch];
#pragma unroll
            for (int i = 0; i < kMoveBatch; ++i) {
                const int j = j0 + i * kMoveThreads + threadIdx.x;
                m[i] = 0.f;
                ks[i] = vs[i] = 0;
                to[i] = -1;
                if (j >= keep) continue;
                const int t = kept[j];
                m[i] = mass[t];
                if (a.cache.k_scale == nullptr || t == j) continue;
                const int64_t from = kv8_row(a.cache, b, h, t);
                to[i] = kv8_row(a.cache, b, h, j);
                ks[i] = from < 0 ? 0 : a.cache.k_scale[from];
                vs[i] = from < 0 ? 0 : a.cache.v_scale[from];
            }
#pragma unroll
            for (int i = 0; i < kMoveBatch; ++i) {
                arrived(m[i]);
                arrived(ks[i]);
                arrived(vs[i]);
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kMoveBatch; ++i) {
                const int j = j0 + i * kMoveThreads + threadIdx.x;
                if (j >= keep) continue;
                new_mass[j] = m[i];
                if (to[i] >= 0) {
                    a.cache.k_scale[to[i]] = (uint8_t)ks[i];
                    a.cache.v_scale[to[i]] = (uint8_t)vs[i];
                }
            }
        }
        __syncthreads();  // (every mass is read)
        for (int t = keep + threadIdx.x; t < L; t += kMoveThreads) new_mass[t] = 0.f;
        return;
    }
    if (L <= keep) return;
    const bool is_v = slice >= a.slices;
    uint8_t* const rows = is_v ? a.cache.v : a.cache.k;
    const int words = a.row_bytes / 16 / a.slices;  // of a row's slice: a power of two
    const int at = 16 * (words * (slice - (is_v ? a.slices : 0)) + (int)threadIdx.x % words);
    const int row_step = kMoveThreads / words, first = threadIdx.x / words;
    const int batch_rows = row_step * kMoveBatch;
    struct Batch {
        u32x4 w[kMoveBatch];
        int64_t to[kMoveBatch];
    };
    auto load = [&](int j0, Batch& x) __attribute__((always_inline)) {
        int t[kMoveBatch];
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i) {
            const int j = j0 + i * row_step + first;
            t[i] = j < keep ? kept[j] : j;
        }
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i) {
            const int j = j0 + i * row_step + first;
            x.to[i] = -1;
            x.w[i] = u32x4{0u, 0u, 0u, 0u};
            if (t[i] == j) continue;  // stays where it is
            const int64_t from = kv8_row(a.cache, b, h, t[i]);
            x.to[i] = kv8_row(a.cache, b, h, j);
            if (from >= 0) x.w[i] = *reinterpret_cast<const u32x4*>(rows + from * a.row_bytes + at);
        }
    };
    auto store = [&](Batch& x) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i) arrived(x.w[i]);
        __builtin_amdgcn_s_barrier();  // the batch is read by all
        asm volatile("" ::: "memory");
#pragma unroll
        for (int i = 0; i < kMoveBatch; ++i)
            if (x.to[i] >= 0) *reinterpret_cast<u32x4*>(rows + x.to[i] * a.row_bytes + at) = x.w[i];
    };
    Batch x, y;
    load(0, x);
    for (int j0 = 0; j0 < keep; j0 += 2 * batch_rows) {
        load(j0 + batch_rows, y);
        store(x);
        load(j0 + 2 * batch_rows, x);
        store(y);
    }
}

}  // namespace

hipError_t launch_evict_select(const EvictArgs& a, const Launch& l) {
    return launch_kernel(evict_select_kernel, wide_grid((int64_t)a.batch * a.cache.n_kv_heads), dim3(kSelectThreads), l, a);
}

// Rows go in slices of a whole line (128 bytes), or in halves of one while those do not make a work-group for every second
// CU.  With 8 kv heads of 8192 rows of 256 bytes, 2048 kept: whole lines against halves 29 -> 38 us for eight sequences,
// 14.8 -> 20.3 for four, but 12.7 -> 10.8 for two.
hipError_t launch_evict_move(const EvictArgs& from, int n_cu, const Launch& l) {
    EvictArgs a = from;
    const int64_t units = (int64_t)a.batch * a.cache.n_kv_heads;
    a.slices = a.row_bytes > 128 ? a.row_bytes / 128 : 1;
    while (a.row_bytes / a.slices > 64 && units * 2 * a.slices < n_cu / 2) a.slices *= 2;
    const int64_t wgs = units * (2 * a.slices + 1);
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    return launch_kernel(evict_move_kernel, wide_grid(wgs), dim3(kMoveThreads), l, a);
}

}  // namespace lara
