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
// the sum is free), and the group's query heads are the 16 rows of operand A, so nothing passes through LDS.  K bounds it: 64
// sequences of 4000 .. 8192 keys of 8 kv heads of 128 take 137-139 us beside other launches (6.0 TB/s) and 133 alone; of the
// E4M3 cache 87 (half the bytes, 5.0 TB/s).
// A block of query rows: a wave keeps 32 or 64 keys as operand B and the rows stream through LDS for the work-group's four
// waves, 32 at a time; rows are shared out over several work-groups where the keys alone do not fill the GPU, and their
// sums meet in a second launch, in a fixed order.  Exponentials beside the products bound it, while other launches fill what a
// wave's chain leaves: 22.0-22.6 us for 2048 causal rows of 32 heads of 128 over 8 kv heads (760-780 TFLOP/s), 5.7 for the last
// 64 rows behind 8192 keys.  Alone, as one engine's calls follow each other, the chain and the shares' uneven lengths bound it:
// 32.5 and 5.1 for the sum (460 TFLOP/s), and 13.9.  The E4M3 cache, whose
// keys are converted once, takes as long: on one stream 33.8 us for 33.2, and 13.5 for 13.3.
#include "decode_common.h"
#include "kv8_device.h"

#include <type_traits>

namespace lara {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kMassWaves = 4;
constexpr int kMassWgs = 32;  // work-groups a CU, of a step

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

// Lanes m and m + 8 of a row of 16 add up: the lane's own value and the other's.
__device__ __forceinline__ float add_far(float own, float far) {
    return own + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(far), 0x128, 0xF, 0xF, true));  // row_ror:8
}

// One row of every sequence.  A work-group: pieces part, part + parts .. of `chunk` keys (a multiple of 256) of one (sequence,
// kv head), rounds of 64 for its waves in turn.
// Rows are loaded by whole lines: lane (m, g) has the 16-byte chunk 4 (m / 8) + g of a line of key m % 8, so an instruction
// covers 8 lines.  A column of operand B is then half of a key's line, and is multiplied with both halves' dims of Q; of the
// two products lanes below 8 keep the first's and add what the lanes above have of theirs.  (16 keys an instruction, half a
// line each: 4.5 TB/s.)  Rows of 64 bytes lie as they are wanted.
template <int D, bool E4M3>
__global__ __launch_bounds__(kMassWaves * 64) void mass_step_kernel(MassArgs a) {
    constexpr int BYTES = E4M3 ? D : 2 * D;
    constexpr bool HALVES = BYTES >= 128;
    constexpr int LOADS = BYTES / 16;           // 16-byte chunks per lane of 64 keys, and per key
    constexpr int PARTS = E4M3 ? 2 : 1;         // steps of 32 dims in a chunk of every lane
    constexpr int STEPS = D / 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m = lane & 15, g = lane >> 4;
    const bool low = m < 8;
    // Pieces go slowest: consecutive work-groups (XCDs in turn) take different sequences and heads, and not always the same
    // piece, of which the later ones are few where lengths differ (64 sequences of 4000 .. 8192 keys: 156 -> 137 us).
    const uint32_t block = wide_block(), units = (uint32_t)a.batch * a.cache.n_kv_heads;
    const int part = block / units, unit = block - part * units;
    const int b = unit / a.cache.n_kv_heads, h = unit - b * a.cache.n_kv_heads;
    if (part >= a.parts) return;
    const int L = clamp_len(a.lens[b], a.cache.l_max);
    if ((int64_t)part * a.chunk >= L) return;
    const int H_q = a.cache.n_kv_heads * a.group;

    // Load i: rows of eight x = i / lines, line i % lines (or 16 rows i, whole).
    constexpr int LINES = HALVES ? BYTES / 128 : 1;
    const uint32_t lane_at = HALVES ? (m & 7) * BYTES + 16 * (4 * (m >> 3) + g) : m * BYTES + 16 * g;
    auto load = [&](int key0, u32x4 (&k)[LOADS], float (&scale)[4], bool* mapped) __attribute__((always_inline)) {
        int64_t row = first_row(a.cache, b, h, key0);
        *mapped = row >= 0;
        if (row < 0) row = 0;
        const uint8_t* const p = a.cache.k + row * BYTES;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(
                p + lane_at + (HALVES ? i / LINES * 8 * BYTES + i % LINES * 128 : i * 16 * BYTES)));
        if constexpr (E4M3)
#pragma unroll
            for (int t = 0; t < 4; ++t) scale[t] = kv8_scale(a.cache.k_scale[row + 16 * t + m]);
    };
    u32x4 k[LOADS];
    float scale[4];
    bool mapped = false;
    int64_t at = (int64_t)part * a.chunk + 64 * wave;
    // The wave's next 64 keys: of the piece, or of the next one.
    auto behind = [&](int64_t key) __attribute__((always_inline)) {
        key += 64 * kMassWaves;
        return ((key - 64 * wave) & (a.chunk - 1)) != 0 ? key : key + (int64_t)(a.parts - 1) * a.chunk;
    };
    if (at < L) load((int)at, k, scale, &mapped);

    // Operand A for step s: the dims that lane (m, g) of the keys holds there, head m.  Chunk c of a row is 16 bytes.
    u32x4 q[STEPS];
    const u32x4* const qp = reinterpret_cast<const u32x4*>(a.q + ((size_t)b * H_q + h * a.group + (m < a.group ? m : 0)) * D);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) q[s] = m < a.group ? qp[PARTS * (g + 4 * (s / PARTS)) + s % PARTS] : u32x4{0u, 0u, 0u, 0u};
    float shift[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = 4 * g + i;
        shift[i] = r < a.group ? row_shift(a.lse[(size_t)b * H_q + h * a.group + r]) : INFINITY;
    }
    float* const mass = a.mass + ((size_t)b * a.cache.n_kv_heads + h) * a.mass_ld;
    // A chunk's part as operand B.
    auto operand = [&](const u32x4& w, int part_of) __attribute__((always_inline)) {
        if constexpr (E4M3) return codes_to_bf16x8(w[2 * part_of], w[2 * part_of + 1]);
        else return w;
    };
    for (int64_t next; at < L; at = next) {
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < 4; ++t) {  // 16 keys
            f32x4 s;
            if constexpr (HALVES) {
                f32x4 acc[2][2];  // [eight keys][half of a line]
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    acc[x][0] = acc[x][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int y = 0; y < LINES; ++y)
#pragma unroll
                        for (int u = 0; u < PARTS; ++u) {
                            const u32x4 kb = operand(k[(2 * t + x) * LINES + y], u);
#pragma unroll
                            for (int half = 0; half < 2; ++half)
                                acc[x][half] = mfma16(q[(2 * y + half) * PARTS + u], kb, acc[x][half]);
                        }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = add_far(low ? acc[0][0][i] : acc[1][1][i], low ? acc[1][0][i] : acc[0][1][i]);
            } else {
                s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int u = 0; u < PARTS; ++u) s = mfma16(q[u], operand(k[t], u), s);
            }
            float c = a.scale_log2;
            if constexpr (E4M3) c *= scale[t];
            float p = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // (a row that adds nothing may have scores of NaN)
                const float e = fast_exp2(fmaf(mapped ? s[i] : 0.f, c, -shift[i]));
                p += shift[i] < INFINITY ? e : 0.f;
            }
            p = pair_sum32(pair_sum16(p));
            sum = g == t ? p : sum;
        }
        const int key = (int)at + lane;
        next = behind(at);
        if (next < L) load((int)next, k, scale, &mapped);
        if (key < L) mass[key] = a.decay == 0.f ? sum : fmaf(a.decay, mass[key], sum);
    }
}

// A block of query rows of sequence b: the rows of a kv head's group, [group][q_len] in order, in stages of 32;
// a work-group takes the stages part, part + parts, ... and KT * 32 keys a wave.
template <int D, bool E4M3, int KT>
__global__ __launch_bounds__(kMassWaves * 64, 2) void mass_block_kernel(MassArgs a) {
    constexpr int NCH = D / 8, STEPS = D / 16, KEYS = 32 * KT, ROWS = 32;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    // kv heads in turn over the work-groups (XCDs), so that one's query rows stay in few L2s.
    const uint32_t block = wide_block();
    const int h = block % a.cache.n_kv_heads, rest = block / a.cache.n_kv_heads;
    const int part = rest % a.parts, kblock = rest / a.parts;
    const int wg_key = kblock * KEYS * kMassWaves;
    if (wg_key >= a.kv_len) return;
    const int key0 = wg_key + KEYS * wave;

    __shared__ __attribute__((aligned(16))) u32x4 rows_in[2][ROWS * NCH];
    __shared__ __attribute__((aligned(16))) float shifts[2][ROWS];
    __shared__ int silent[2];  // whether some row of the stage adds nothing

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

    const int rows = a.group * a.q_len, stages = (rows + ROWS - 1) / ROWS;
    const uint16_t* const q = a.q + (size_t)h * rows * D;
    const float* const lse = a.lse + (size_t)h * rows;
    // The last row that sees the work-group's first key decides whether a stage is worked on at all: of one head's rows
    // their last, of several heads' any.
    const int64_t first_seen = (int64_t)a.kv_pos_base + wg_key - a.q_pos_base;  // the least query row that sees wg_key
    auto next_seen = [&](int st) __attribute__((always_inline)) {
        if (a.causal)
            for (; st < stages; st += a.parts) {
                const int i0 = ROWS * st % a.q_len, n = min(ROWS, rows - ROWS * st);
                if ((int64_t)min(i0 + n, a.q_len) > first_seen) break;
            }
        return st;
    };
    constexpr int THREADS = kMassWaves * 64, PER = ROWS * NCH / THREADS;  // 16-byte chunks of a stage per thread
    static_assert(PER >= 1, "a stage is a load a thread at least");
    u32x4 in[PER];
    float in_lse = 0.f;
    auto load = [&](int st) __attribute__((always_inline)) {
        const u32x4* const from = reinterpret_cast<const u32x4*>(q) + (size_t)ROWS * st * NCH;
        const int n = rows - ROWS * st;  // rows left
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int slot = i * THREADS + threadIdx.x;
            in[i] = slot / NCH < n ? from[slot] : u32x4{0u, 0u, 0u, 0u};
        }
        if (threadIdx.x < ROWS) in_lse = (int)threadIdx.x < n ? lse[ROWS * st + threadIdx.x] : INFINITY;  // (worked on as it is stored)
    };
    float sum[KT];
#pragma unroll
    for (int t = 0; t < KT; ++t) sum[t] = 0.f;
    const int64_t sees = (int64_t)a.kv_pos_base + key0 - a.q_pos_base;  // the least query row that sees the wave's first key
    const int first_row = !a.causal ? -(1 << 30) : (int)(sees < -(1 << 30) ? -(1 << 30) : sees) + col;
    int st = next_seen(part), at = 0;
    if (st < stages) load(st);
    for (; st < stages; at ^= 1) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int slot = i * THREADS + threadIdx.x, r = slot / NCH, c = slot % NCH;
            rows_in[at][r * NCH + (c ^ (NCH == 16 ? r & 15 : (r >> 1) & 7))] = in[i];
        }
        if (threadIdx.x < ROWS) {
            const float shift = row_shift(in_lse);
            shifts[at][threadIdx.x] = shift;
            silent[at] = __ballot(shift == INFINITY) != 0;
        }
        const int next = next_seen(st + a.parts);
        if (next < stages) load(next);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the stage is written; the loads stay in flight
        __builtin_amdgcn_s_barrier();  // (two stages: the one before is read by now, or will not be written before the next barrier)
        asm volatile("" ::: "memory");
        // Whether some row of the stage does not see some key of the wave.
        const int i0 = ROWS * st % a.q_len;
        const bool several = i0 + ROWS > a.q_len;
        const bool mask = a.causal && (several || i0 < sees + KEYS - 1);
        const int silence = silent[at];
        f32x16 acc[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[kt][i] = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const u32x4 qa = rows_in[at][col * NCH + ((2 * s + half) ^ (NCH == 16 ? col & 15 : (col >> 1) & 7))];
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) acc[kt] = mfma32(qa, k[kt][s], acc[kt]);
        }
        auto add = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4) {
                const f32x4 shift = *reinterpret_cast<const f32x4*>(&shifts[at][8 * i4 + 4 * half]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    int row = i0 + 8 * i4 + 4 * half + i;
                    if (masked && several) row %= a.q_len;
                    if (masked) row = shift[i] == INFINITY ? INT_MIN : row;  // (it adds nothing, whatever its scores)
#pragma unroll
                    for (int kt = 0; kt < KT; ++kt) {
                        const float p = fast_exp2(fmaf(acc[kt][4 * i4 + i], scale[kt], -shift[i]));
                        sum[kt] += masked && row < first_row + 32 * kt ? 0.f : p;
                    }
                }
            }
        };
        if (((mask ? 1 : 0) | __builtin_amdgcn_readfirstlane(silence)) != 0) add(std::true_type{});
        else add(std::false_type{});
        st = next;
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

// Work-groups of a step: pieces of 512 keys, or 256 while those do not make four work-groups a CU; 32 work-groups a CU at most,
// which take the pieces in turn, so that a context's capacity does not cost what it does not hold (64 sequences of
// 1000 keys in contexts of 131072, 8 kv heads: 78 -> 24.5 us).
hipError_t launch_mass_step(int head_dim, MassArgs a, int n_cu, const Launch& l) {
    const int64_t units = (int64_t)a.batch * a.cache.n_kv_heads;
    a.chunk = 512;
    while (a.chunk > 256 && units * ((a.cache.l_max + a.chunk - 1) / a.chunk) < 4 * n_cu) a.chunk /= 2;
    a.parts = (int)std::min<int64_t>(((int64_t)a.cache.l_max + a.chunk - 1) / a.chunk, std::max<int64_t>(1, kMassWgs * n_cu / units));
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
    p.key_tiles = kv_len > 128 ? 2 : 1;
    const int64_t keys = 32 * p.key_tiles * kMassWaves, of_keys = n_kv_heads * ((kv_len + keys - 1) / keys);
    // A few stages on every CU are sooner done than shared out and summed by a second launch.  One launch against two, 64 rows of
    // 4 heads (8 stages) of 8 kv heads at the end of 8192 keys: 5.8 us against 7.1 beside other launches, 13.3 / 13.5 on one
    // stream.  (Below the border, 7168 keys, 5.7 / 6.7 and 13.3 / 13.5, 4200 keys 4.9 / 6.5 and 12.7 / 12.9: it could be lower.)
    if (of_keys >= n_cu && tiles <= 16)
        p.parts = 1;
    else  // (a prompt of 2048 rows and 32 heads: 3 work-groups a CU, which all are on it at once, 21.9 us; 4 of them 22.9)
        p.parts = (int)std::max<int64_t>(1, std::min<int64_t>({kMassBlockWgs * n_cu / of_keys, (int64_t)tiles / 4, kMassMaxParts}));
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
