// The attention weight that every cache row gets.  With the log-sum-exp of a query row's scaled scores, as attention
// returns it,
//   p_rt = exp(scale * q_r . k_t - lse_r)      mass_t = decay * mass_t + sum over the query rows r that see t of p_rt
// per kv head, over the query heads of its group (and the rows of a block of queries).  V is not read.
//
// The scores are S = Q . K^T on the matrix cores, keys as columns: a lane holds several rows of one key, so the sum over
// rows is additions in the lane, and the rows' maximum is not needed (lse stands for it: no p is above 1 but for rounding).
// p, the sums and the mass are fp32.  A row whose lse is not finite (it has no keys, or a NaN among its scores) adds nothing.
//
// One row of every sequence: a wave loads 64 keys, whose 16-byte chunks are operand B as they lie (the order of the dims in
// the sum is free), and the group's query heads are the 16 rows of operand A, so nothing passes through LDS.
// A block of query rows: a wave keeps 32 or 64 keys as operand B and the rows stream through LDS for the work-group's four
// waves, 32 at a time; rows are shared out over several work-groups where the keys alone do not fill the GPU, and their
// sums meet in a second launch, in a fixed order.
#include "decode_common.h"
#include "kv8_device.h"

namespace lara {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMassWaves = 4;

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Eight codes as bf16 (exact); the row's scale multiplies the score.
__device__ __forceinline__ u32x4 codes_to_bf16x8(uint32_t lo, uint32_t hi) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true))};
}

// What is subtracted from a row's scores (log2 units): infinite for a row that adds nothing.
__device__ __forceinline__ float row_shift(float lse) { return fabsf(lse) < INFINITY ? lse * (1.0f / kLn2) : INFINITY; }

// The row of a sequence's kv head at which 64 keys from key0 (a multiple of 64) lie, or -1: unmapped (rows of zeros).
__device__ __forceinline__ int64_t first_row(const Kv8Cache& c, int b, int h, int key0) {
    if (c.block_table == nullptr) return ((int64_t)b * c.n_kv_heads + h) * c.l_cap + key0;
    return paged_row_uniform(c.block_table + (size_t)b * c.max_pages, c.page_shift, c.n_kv_heads, h, key0);
}

// One row of every sequence.  A work-group: `chunk` keys (a multiple of 256) of one (sequence, kv head), rounds of 64 for
// its waves in turn.
template <int D, bool E4M3>
__global__ __launch_bounds__(kMassWaves * 64) void mass_step_kernel(MassArgs a) {
    constexpr int CH = E4M3 ? D / 64 : D / 32;  // 16-byte chunks of a key per lane
    constexpr int BYTES = E4M3 ? D : 2 * D;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4;
    const uint32_t block = wide_block();
    const int unit = block / a.parts, part = block - unit * a.parts;
    const int b = unit / a.cache.n_kv_heads, h = unit - b * a.cache.n_kv_heads;
    if (b >= a.batch) return;
    const int L = clamp_len(a.lens[b], a.cache.l_max);
    const int64_t begin = (int64_t)part * a.chunk;
    if (begin >= L) return;
    const int end = begin + a.chunk < L ? (int)(begin + a.chunk) : L;
    const int H_q = a.cache.n_kv_heads * a.group;

    auto load = [&](int key0, u32x4 (&k)[4][CH], float (&scale)[4], bool* mapped) __attribute__((always_inline)) {
        int64_t row = first_row(a.cache, b, h, key0);
        *mapped = row >= 0;
        if (row < 0) row = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint8_t* const p = a.cache.k + (row + 16 * t + m) * BYTES + 16 * g;
#pragma unroll
            for (int j = 0; j < CH; ++j) k[t][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + 64 * j));
            if constexpr (E4M3) scale[t] = kv8_scale(a.cache.k_scale[row + 16 * t + m]);
        }
    };
    u32x4 k[4][CH];
    float scale[4];
    bool mapped = false;
    int key0 = (int)begin + 64 * wave;
    if (key0 < end) load(key0, k, scale, &mapped);

    // Operand A: lane (m, g) holds, for chunk j, the dims that the lanes of the keys hold there.
    constexpr int STEPS = D / 32;
    u32x4 q[STEPS];
    const u32x4* const qp = reinterpret_cast<const u32x4*>(a.q + ((size_t)b * H_q + h * a.group + (m < a.group ? m : 0)) * D);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) q[s] = m < a.group ? qp[E4M3 ? 2 * (g + 4 * (s >> 1)) + (s & 1) : g + 4 * s] : u32x4{0u, 0u, 0u, 0u};
    float shift[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * g + i;
        shift[i] = r < a.group ? row_shift(a.lse[(size_t)b * H_q + h * a.group + r]) : INFINITY;
    }
    float* const mass = a.mass + ((size_t)b * a.cache.n_kv_heads + h) * a.mass_ld;
    for (; key0 < end; key0 += 64 * kMassWaves) {
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                u32x4 kb;
                if constexpr (E4M3) {
                    const u32x4& w = k[t][s >> 1];
                    kb = codes_to_bf16x8(w[2 * (s & 1)], w[2 * (s & 1) + 1]);
                } else {
                    kb = k[t][s];
                }
                acc = mfma16(q[s], kb, acc);
            }
            float c = a.scale_log2;
            if constexpr (E4M3) c *= scale[t];
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) p += fast_exp2(fmaf(mapped ? acc[i] : 0.f, c, -shift[i]));
            p = pair_sum32(pair_sum16(p));
            sum = g == t ? p : sum;
        }
        const int key = key0 + lane;
        const int next = key0 + 64 * kMassWaves;
        if (next < end) load(next, k, scale, &mapped);
        if (key < end) mass[key] = a.decay == 0.f ? sum : fmaf(a.decay, mass[key], sum);
    }
}

// A block of query rows of sequence b: the rows of a kv head's group, [group][q_len] in order, in tiles of 32; a work-group
// takes the tiles part, part + parts, ... and KT * 32 keys a wave.
template <int D, bool E4M3, int KT>
__global__ __launch_bounds__(kMassWaves * 64, 2) void mass_block_kernel(MassArgs a) {
    constexpr int NCH = D / 8, STEPS = D / 16, KEYS = 32 * KT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    // kv heads in turn over the work-groups (XCDs), so that one's query rows stay in few L2s.
    const uint32_t block = wide_block();
    const int h = block % a.cache.n_kv_heads, rest = block / a.cache.n_kv_heads;
    const int part = rest % a.parts, kblock = rest / a.parts;
    const int wg_key = kblock * KEYS * kMassWaves;
    if (wg_key >= a.kv_len) return;
    const int key0 = wg_key + KEYS * wave;

    __shared__ __attribute__((aligned(16))) u32x4 tile[2][32 * NCH];
    __shared__ __attribute__((aligned(16))) float shifts[2][32];

    // Operand B: lane l keeps dims 16 s + 8 (l / 32) .. of key l % 32 of each tile.
    u32x4 k[KT][STEPS];
    float scale[KT];
    bool there[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const int key = key0 + 32 * t + col;
        there[t] = key < a.kv_len;
        const int64_t row = there[t] ? kv8_row(a.cache, a.b, h, key) : -1;
        const uint8_t* const p = a.cache.k + (row < 0 ? 0 : row) * (E4M3 ? D : 2 * D);
        scale[t] = a.scale_log2;
        if constexpr (E4M3) scale[t] *= row < 0 ? 0.f : kv8_scale(a.cache.k_scale[row]);
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            if constexpr (E4M3) {
                const u32x2 w = reinterpret_cast<const u32x2*>(p)[2 * s + half];
                k[t][s] = codes_to_bf16x8(w[0], w[1]);
            } else {
                k[t][s] = reinterpret_cast<const u32x4*>(p)[2 * s + half];
            }
            if (row < 0) k[t][s] = u32x4{0u, 0u, 0u, 0u};
        }
    }

    const int rows = a.group * a.q_len, tiles = (rows + 31) / 32;
    const uint16_t* const q = a.q + (size_t)h * rows * D;
    const float* const lse = a.lse + (size_t)h * rows;
    // The last row position that sees the work-group's first key decides whether a tile is worked on at all: of one head,
    // its last row; of two, both ends.
    const int64_t first_seen = (int64_t)a.kv_pos_base + wg_key - a.q_pos_base;  // the least query row that sees wg_key
    auto seen = [&](int t) __attribute__((always_inline)) {
        if (!a.causal) return true;
        const int r0 = 32 * t, r1 = min(r0 + 31, rows - 1);
        const int i0 = r0 % a.q_len, i1 = r1 % a.q_len;
        return (r1 - r0 != i1 - i0 ? (int64_t)a.q_len - 1 : (int64_t)i1) >= first_seen;
    };
    constexpr int PER = 32 * NCH / (kMassWaves * 64);  // 16-byte chunks of a tile per thread
    static_assert(PER >= 1, "a tile is a load a thread at least");
    u32x4 in[PER];
    float in_shift = INFINITY;
    auto load = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int slot = i * kMassWaves * 64 + threadIdx.x, r = 32 * t + slot / NCH;
            in[i] = r < rows ? reinterpret_cast<const u32x4*>(q)[(size_t)r * NCH + slot % NCH] : u32x4{0u, 0u, 0u, 0u};
        }
        if (threadIdx.x < 32) {
            const int r = 32 * t + threadIdx.x;
            in_shift = r < rows ? row_shift(lse[r]) : INFINITY;
        }
    };
    auto next_seen = [&](int t) __attribute__((always_inline)) {
        while (t < tiles && !seen(t)) t += a.parts;
        return t;
    };
    float sum[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) sum[t] = 0.f;
    int t = next_seen(part), at = 0;
    if (t < tiles) load(t);
    for (; t < tiles; at ^= 1) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int slot = i * kMassWaves * 64 + threadIdx.x, r = slot / NCH, c = slot % NCH;
            tile[at][r * NCH + (c ^ (NCH == 16 ? r & 15 : (r >> 1) & 7))] = in[i];
        }
        if (threadIdx.x < 32) shifts[at][threadIdx.x] = in_shift;
        const int next = next_seen(t + a.parts);
        if (next < tiles) load(next);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the tile is written; the loads stay in flight
        __builtin_amdgcn_s_barrier();  // (two tiles: the one before is read by now, or will not be written before the next barrier)
        asm volatile("" ::: "memory");
        const int i0 = 32 * t % a.q_len;
        f32x16 acc[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[kt][i] = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const u32x4 qa = tile[at][col * NCH + ((2 * s + half) ^ (NCH == 16 ? col & 15 : (col >> 1) & 7))];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) acc[kt] = mfma32(qa, k[kt][s], acc[kt]);
        }
        // Whether some row of the tile does not see some key of the wave.
        const bool mask = a.causal && (i0 + 31 >= a.q_len || (int64_t)i0 + a.q_pos_base < (int64_t)a.kv_pos_base + key0 + KEYS - 1);
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
            const f32x4 shift = *reinterpret_cast<const f32x4*>(&shifts[at][8 * i4 + 4 * half]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    float p = fast_exp2(fmaf(acc[kt][4 * i4 + i], scale[kt], -shift[i]));
                    if (mask) {
                        const int r = (32 * t + 8 * i4 + 4 * half + i) % a.q_len;
                        if ((int64_t)r + a.q_pos_base < (int64_t)a.kv_pos_base + key0 + 32 * kt + col) p = 0.f;
                    }
                    sum[kt] += p;
                }
            }
        }
        t = next;
    }
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        const float p = pair_sum32(sum[kt]);
        const int key = key0 + 32 * kt + col;
        if (half != 0 || !there[kt]) continue;
        if (a.parts > 1) {
            a.part_sums[((size_t)part * a.cache.n_kv_heads + h) * a.kv_len + key] = p;
        } else {
            float* const to = a.mass + ((size_t)a.b * a.cache.n_kv_heads + h) * a.mass_ld + key;
            *to = a.decay == 0.f ? p : fmaf(a.decay, *to, p);
        }
    }
}

__global__ __launch_bounds__(256) void mass_sum_kernel(MassArgs a) {
    const int64_t i = (int64_t)wide_block() * 256 + threadIdx.x;
    const int64_t n = (int64_t)a.cache.n_kv_heads * a.kv_len;
    if (i >= n) return;
    float sum = 0.f;
    for (int p = 0; p < a.parts; ++p) sum += a.part_sums[p * n + i];
    const int h = (int)(i / a.kv_len);
    float* const to = a.mass + ((size_t)a.b * a.cache.n_kv_heads + h) * a.mass_ld + (i - (int64_t)h * a.kv_len);
    *to = a.decay == 0.f ? sum : fmaf(a.decay, *to, sum);
}

}  // namespace

// Work-groups of a step: pieces of 1024 keys, or fewer down to 256 while those do not make four work-groups a CU.
hipError_t launch_mass_step(int head_dim, MassArgs a, int n_cu, const Launch& l) {
    const int64_t units = (int64_t)a.batch * a.cache.n_kv_heads;
    a.chunk = 1024;
    while (a.chunk > 256 && units * ((a.cache.l_max + a.chunk - 1) / a.chunk) < 4 * n_cu) a.chunk /= 2;
    a.parts = (a.cache.l_max + a.chunk - 1) / a.chunk;
    const int64_t wgs = units * a.parts;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid = wide_grid(wgs), block(kMassWaves * 64);
    const bool e4m3 = a.cache.k_scale != nullptr;
    if (head_dim == 128)
        return e4m3 ? launch_kernel(mass_step_kernel<128, true>, grid, block, l, a) : launch_kernel(mass_step_kernel<128, false>, grid, block, l, a);
    if (head_dim == 64)
        return e4m3 ? launch_kernel(mass_step_kernel<64, true>, grid, block, l, a) : launch_kernel(mass_step_kernel<64, false>, grid, block, l, a);
    return hipErrorInvalidValue;
}

MassPlan plan_mass_block(int group, int n_kv_heads, int q_len, int kv_len, int n_cu) {
    const int tiles = (int)(((int64_t)group * q_len + 31) / 32);
    MassPlan p;
    p.key_tiles = 2;
    auto wgs = [&](int kt) { return (int64_t)n_kv_heads * ((kv_len + 128 * kt - 1) / (128 * kt)); };
    if (wgs(2) < 2 * n_cu) p.key_tiles = 1;
    const int64_t of_keys = wgs(p.key_tiles);
    p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({4 * n_cu / of_keys, (int64_t)tiles / 4, kMassMaxParts}));
    return p;
}

template <int D, bool E4M3>
static hipError_t launch_mass_block_t(const MassArgs& a, int key_tiles, const Launch& l) {
    const int keys = 32 * key_tiles * kMassWaves;
    const int64_t wgs = (int64_t)a.cache.n_kv_heads * a.parts * ((a.kv_len + keys - 1) / keys);
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid = wide_grid(wgs), block(kMassWaves * 64);
    return key_tiles == 2 ? launch_kernel(mass_block_kernel<D, E4M3, 2>, grid, block, l, a) : launch_kernel(mass_block_kernel<D, E4M3, 1>, grid, block, l, a);
}

hipError_t launch_mass_block(int head_dim, const MassArgs& a, int key_tiles, const Launch& l) {
    const bool e4m3 = a.cache.k_scale != nullptr;
    if (head_dim == 128) return e4m3 ? launch_mass_block_t<128, true>(a, key_tiles, l) : launch_mass_block_t<128, false>(a, key_tiles, l);
    if (head_dim == 64) return e4m3 ? launch_mass_block_t<64, true>(a, key_tiles, l) : launch_mass_block_t<64, false>(a, key_tiles, l);
    return hipErrorInvalidValue;
}

hipError_t launch_mass_sum(const MassArgs& a, const Launch& l) {
    const int64_t wgs = ((int64_t)a.cache.n_kv_heads * a.kv_len + 255) / 256;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    return launch_kernel(mass_sum_kernel, wide_grid(wgs), dim3(256), l, a);
}

}  // namespace lara
