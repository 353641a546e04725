// Eviction from the cache: of every (sequence, kv head) with more than `keep` rows the first `sinks`, the last `recent` and
// the heaviest between stay, by the mass that they have; equal ones go by their index, NaN counts as less than anything.
// The rows that stay move together, in their order, to the first `keep`.
//
// Selection, a work-group per (sequence, kv head): the least mass that stays is found by its bits, 11, 11 and 10 at a time
// (masses as unsigned numbers of the same order; a histogram of the masses that share the bits found so far).  Then the rows
// are counted by 64, which gives every row that stays its place.
//
// Moving, in place: row j comes from row kept[j] >= j, and kept rises, so a work-group that takes the rows in order, a batch
// at a time, has read all that a batch's stores may overwrite once the batch itself is read; the next batch's loads may even
// pass them.  Rows do not mix along their bytes, so a (sequence, kv head) is shared out by K and V and by columns, which
// need nothing of each other: no work-group waits for another.  Scales and masses are one more work-group's.
#include "decode_common.h"
#include "kv8_device.h"

namespace lara {
namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kSelectHeld = 16;  // masses a thread keeps in registers; those past them are read again
constexpr int kBins = 2048;
constexpr int kMoveThreads = 256, kMoveBatch = 8;  // 16-byte words of a batch per thread

// The order of masses as that of unsigned numbers: NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t mass_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictArgs a) {
    const int unit = wide_block(), b = unit / a.cache.n_kv_heads;
    if (b >= a.batch) return;
    const int L = clamp_len(a.lens[b], a.cache.l_max), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (unit == b * a.cache.n_kv_heads && tid == 0) a.lens_copy[b] = L;
    int32_t* const kept = a.kept + (size_t)unit * a.keep;
    if (L <= a.keep) {
        for (int j = tid; j < a.keep; j += kSelectThreads) kept[j] = j < L ? j : -1;
        return;
    }
    const float* const mass = a.mass + (size_t)unit * a.mass_ld;
    const int lo = a.sinks, hi = L - a.recent, need = a.keep - a.sinks - a.recent;
    uint32_t held[kSelectHeld];
#pragma unroll
    for (int c = 0; c < kSelectHeld; ++c) {
        const int t = c * kSelectThreads + tid;
        held[c] = t >= lo && t < hi ? mass_key(mass[t]) : 0u;
    }
    // Calls f(row, key) for the thread's rows of the middle.
    auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < kSelectHeld; ++c) {
            const int t = c * kSelectThreads + tid;
            if (t >= lo && t < hi) f(held[c]);
        }
        for (int t = kSelectHeld * kSelectThreads + tid; t < hi; t += kSelectThreads)
            if (t >= lo) f(mass_key(mass[t]));
    };
    __shared__ int hist[kBins];
    __shared__ int wave_total[kSelectWaves];
    __shared__ int found[2];
    uint32_t least = 0xFFFFFFFFu, mask = 0;  // (no mass has that key: nothing of the middle stays where need is 0)
    int quota = 0;                           // rows that stay of those with the least key
    if (need > 0) {
        least = 0;
        quota = need;
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
            for (int i = tid; i < kBins; i += kSelectThreads) hist[i] = 0;
            __syncthreads();
            each([&](uint32_t k) {
                if ((k & mask) == least) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
            });
            __syncthreads();
            // Bins from the top: thread t has two of them; the one in which the count reaches the quota is it.
            const int top = bins - 1 - 2 * tid;
            const int n0 = top >= 0 ? hist[top] : 0, n1 = top >= 1 ? hist[top - 1] : 0;
            const int upto = wave_scan(n0 + n1);
            if (lane == 63) wave_total[wave] = upto;
            __syncthreads();
            int before = upto - n0 - n1;
            for (int w = 0; w < wave; ++w) before += wave_total[w];
            if (before < quota && quota <= before + n0 + n1) {
                const bool second = quota > before + n0;
                found[0] = top - (second ? 1 : 0);
                found[1] = quota - before - (second ? n0 : 0);
            }
            __syncthreads();
            least |= (uint32_t)found[0] << shift;
            mask |= (uint32_t)(bins - 1) << shift;
            quota = found[1];
        }
    }
    // Places, 256 runs of 64 rows at a time: run 16 c + w is wave w's.
    __shared__ int sure_of[16 * kSelectWaves], even_of[16 * kSelectWaves];
    __shared__ int scan_total[4][2];
    int sure_before = 0, even_before = 0;
    for (int t0 = 0; t0 < L; t0 += 16 * kSelectThreads) {
        unsigned long long sure[16], even[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            const int t = t0 + c * kSelectThreads + tid;
            const bool middle = t >= lo && t < hi;
            const uint32_t k = t0 == 0 ? held[c] : middle ? mass_key(mass[t]) : 0u;
            sure[c] = __ballot(t < L && (!middle || k > least));
            even[c] = __ballot(middle && k == least);
            if (lane == 0) {
                sure_of[c * kSelectWaves + wave] = __popcll(sure[c]);
                even_of[c * kSelectWaves + wave] = __popcll(even[c]);
            }
        }
        __syncthreads();
        int s = 0, e = 0, s_upto = 0, e_upto = 0;
        if (wave < 4) {
            s = sure_of[tid];
            e = even_of[tid];
            s_upto = wave_scan(s);
            e_upto = wave_scan(e);
            if (lane == 63) {
                scan_total[wave][0] = s_upto;
                scan_total[wave][1] = e_upto;
            }
        }
        __syncthreads();
        if (wave < 4) {
            int sb = sure_before, eb = even_before;
            for (int w = 0; w < wave; ++w) {
                sb += scan_total[w][0];
                eb += scan_total[w][1];
            }
            sure_of[tid] = sb + s_upto - s;
            even_of[tid] = eb + e_upto - e;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            const int t = t0 + c * kSelectThreads + tid;
            const unsigned long long below = (1ull << lane) - 1;
            const int e_rank = even_of[c * kSelectWaves + wave] + __popcll(even[c] & below);
            const int place = sure_of[c * kSelectWaves + wave] + __popcll(sure[c] & below) + min(e_rank, quota);
            const bool stays = (sure[c] >> lane & 1) != 0 || ((even[c] >> lane & 1) != 0 && e_rank < quota);
            if (stays) kept[place] = t;
        }
        for (int w = 0; w < 4; ++w) {
            sure_before += scan_total[w][0];
            even_before += scan_total[w][1];
        }
        __syncthreads();  // the counts are read
    }
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

// Rows go in slices of a whole line (128 bytes), or finer ones down to 32 bytes while those do not make two work-groups a CU.
hipError_t launch_evict_move(const EvictArgs& from, int n_cu, const Launch& l) {
    EvictArgs a = from;
    const int64_t units = (int64_t)a.batch * a.cache.n_kv_heads;
    a.slices = a.row_bytes > 128 ? a.row_bytes / 128 : 1;
    while (a.row_bytes / a.slices > 32 && units * 2 * a.slices < 2 * n_cu) a.slices *= 2;
    const int64_t wgs = units * (2 * a.slices + 1);
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    return launch_kernel(evict_move_kernel, wide_grid(wgs), dim3(kMoveThreads), l, a);
}

}  // namespace lara
