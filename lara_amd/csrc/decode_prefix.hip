// Decode for a batch that shares a prefix: sequence b attends the first shared[b] rows of sequence prefix_b and then its own
// lens[b] rows, as one softmax,
//   o = sum over both of p_k v_k / sum of p_k,   p_k = exp(scale * q . k_k - m),
// and every row of the prefix is read for the whole batch, not once per sequence.
//
// The prefix's keys are cut into pieces and its query rows -- those of all sequences and of a kv head's group, [b][g] --
// into blocks of 32 * row_tiles; a work-group has a piece and a block.  Own rows are cut into pieces of a power of two keys,
// a wave each.  All leave fp32 partials (O, m, l), which a second launch joins with log-sum-exp weights.  Work-groups of
// both kinds alternate, so that a CU holds some of each: the prefix's are bound by the matrix cores, the others by memory.
//
// One step, for 32 query rows and 32 or 64 keys, in both:
//   S^T [keys x 32 rows] = K . Q^T, O^T [D x 32 rows] += V^T . P^T by v_mfma_f32_32x32x16_bf16, with K and V in LDS (E4M3
// codes are turned to bf16, which holds them, on their way there) and one row's softmax in a lane pair.  Of the work-group's
// four waves row_tiles share a tile of K and V and the others take other tiles of the piece; a wave of own rows has its tile
// to itself.  The next tile's loads are under way while one is computed.
//
// p is rounded to bf16 before the second product (half a step, 2^-8 of it at most), l sums the unrounded ones; scores, sums
// and O are fp32.  A row is 0 (lse -inf) without keys, NaN with a score of NaN.  Rows of V that a sequence does not see do not
// reach it, whatever they hold: past the end they are read as zeros, and where the batch's lengths differ inside a tile with
// infinities or NaN the keys are added one at a time.
#include "decode_common.h"
#include "kv8_device.h"

#include <type_traits>

namespace lara {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;
constexpr int kOwnKeys = 32;  // keys of a step of own rows

__device__ __forceinline__ f32x16 mfma32(const u32x4& a, const u32x4& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}

// Element i % 4 of the 8 bytes that lane 4j + i / 4 of a 16-lane group addresses, j = 0..3, for its lane i.
__device__ __forceinline__ u32x2 lds_read_tr16(const void* p) {
    typedef __attribute__((address_space(3))) i16x4_t lds_i16x4;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p)));
}

// 16-byte chunks of a tile's rows are permuted: K's for reads of one chunk of 32 rows, V's for transposing reads of four.
template <int D>
__device__ __forceinline__ int k_chunk(int row, int c) {
    return c ^ (D == 128 ? row & 15 : (row >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_chunk(int row, int c) {
    return c ^ (D == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1));
}

__device__ __forceinline__ u32x4 codes_to_bf16x8(uint32_t lo, uint32_t hi, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
}

// LDS traffic of the wave is complete; its global loads stay in flight.
__device__ __forceinline__ void lds_done() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void lds_barrier() {
    lds_done();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ---- own rows' pieces ------------------------------------------------------------------------------------

// Lengths of own rows, 64 sequences at a time, one per lane.
__device__ __forceinline__ int own_len(const PrefixArgs& a, int s) { return s < a.batch ? clamp_len(a.lens[s], a.cache.l_max) : 0; }

// Pieces have 2^log2 keys, the least of 64 and more with which they fit the partials and there are at most `most` of
// them -- or one each, which always fits.  (The same for every wave and both launches: it follows from the lengths.)
constexpr int kOwnLog2 = 6;
__device__ __forceinline__ int own_pieces(int len, int log2) { return (len + (1 << log2) - 1) >> log2; }
__device__ __forceinline__ int own_log2(const PrefixArgs& a) {
    const int lane = threadIdx.x & 63;
    const int64_t most = a.own_slots;
    for (int log2 = kOwnLog2; log2 < 30; ++log2) {
        int64_t n = 0;
        for (int c0 = 0; c0 < a.batch; c0 += 64) n += __builtin_amdgcn_readlane(wave_scan(own_pieces(own_len(a, c0 + lane), log2)), 63);
        if (n * a.cache.n_kv_heads <= most) return log2;
    }
    return 30;
}

// ---- one task: 32 query rows over a run of tiles -----------------------------------------------------------

template <int D>
struct Rows {
    u32x4 q[D / 16];
    f32x16 o[D / 32];
    float m, l;
    int limit;  // keys that the lane's row sees
};

template <int D>
__device__ __forceinline__ void rows_clear(Rows<D>& r) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) r.o[t][i] = 0.f;
    r.m = -INFINITY;
    r.l = 0.f;
}

// A tile of NT * 32 keys on its way into LDS through the registers of TEAM waves; `t` is the thread's place among them.
template <int D, bool E4M3, int NT, int TEAM>
struct Staged {
    static constexpr int NCH = D / 8, KEYS = 32 * NT, THREADS = 64 * TEAM;
    static constexpr int PIECES = E4M3 ? D / 16 : NCH;  // 16-byte loads of a row
    static constexpr int N = KEYS * PIECES / THREADS;
    static_assert(N >= 1 && N * THREADS == KEYS * PIECES, "whole loads");
    u32x4 k[N], v[N];
    uint8_t ks[N], vs[N];  // E4M3: scale bytes
    int live;              // rows that hold keys

    __device__ __forceinline__ void load(const PrefixArgs& a, int b, int h, int key0, int end, int t) {
        int64_t row;
        if (a.cache.block_table == nullptr)
            row = ((int64_t)b * a.cache.n_kv_heads + h) * a.cache.l_cap + key0;
        else
            row = paged_row_uniform(a.cache.block_table + (size_t)b * a.cache.max_pages, a.cache.page_shift, a.cache.n_kv_heads, h, key0);
        live = row < 0 ? 0 : end - key0;  // (an unmapped page: rows of zeros, from any that is there)
        if (row < 0) row = 0;
        const u32x4* const kp = reinterpret_cast<const u32x4*>(a.cache.k) + row * PIECES + t;
        const u32x4* const vp = reinterpret_cast<const u32x4*>(a.cache.v) + row * PIECES + t;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            k[i] = kp[i * THREADS];
            v[i] = vp[i * THREADS];
            if constexpr (E4M3) {
                ks[i] = a.cache.k_scale[row + (i * THREADS + t) / PIECES];
                vs[i] = a.cache.v_scale[row + (i * THREADS + t) / PIECES];
            }
        }
    }
    __device__ __forceinline__ void store(u32x4* lk, u32x4* lv, int t) {
        const bool whole = live >= KEYS;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int slot = i * THREADS + t, key = slot / PIECES, c = slot % PIECES;
            const bool there = whole || key < live;
            if constexpr (E4M3) {
                const float kscale = kv8_scale(ks[i]), vscale = kv8_scale(vs[i]);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const u32x4 kw = codes_to_bf16x8(k[i][2 * half], k[i][2 * half + 1], kscale);
                    const u32x4 vw = codes_to_bf16x8(v[i][2 * half], v[i][2 * half + 1], vscale);
                    lk[key * NCH + k_chunk<D>(key, 2 * c + half)] = there ? kw : u32x4{0u, 0u, 0u, 0u};
                    lv[key * NCH + v_chunk<D>(key, 2 * c + half)] = there ? vw : u32x4{0u, 0u, 0u, 0u};
                }
            } else {
                lk[key * NCH + k_chunk<D>(key, c)] = there ? k[i] : u32x4{0u, 0u, 0u, 0u};
                lv[key * NCH + v_chunk<D>(key, c)] = there ? v[i] : u32x4{0u, 0u, 0u, 0u};
            }
        }
    }
};

// The tile of keys key0 .. in LDS, for 32 rows.  UNEVEN: the rows' limits differ.  [lo, hi]: the least and the largest.
template <int D, int NT, bool UNEVEN>
__device__ __forceinline__ void attend(Rows<D>& r, const u32x4* lk, const u32x4* lv, int key0, int lo, float scale_log2) {
    constexpr int NCH = D / 8, STEPS = D / 16, MT = D / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    f32x16 s[NT];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
#pragma unroll
    for (int st = 0; st < STEPS; ++st)
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) {
            const int row = 32 * kt + col;
            s[kt] = mfma32(lk[row * NCH + k_chunk<D>(row, 2 * st + half)], r.q[st], s[kt]);
        }
    const bool mask = key0 + 32 * NT > lo;  // (wave-uniform)
    if (mask) {
#pragma unroll
        for (int kt = 0; kt < NT; ++kt)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[kt][i] = key0 + 32 * kt + 8 * (i >> 2) + 4 * half + (i & 3) < r.limit ? s[kt][i] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kt][i]);
    const float cand = fmaxf(r.m, pair_max32(mx) * scale_log2);
    if (__ballot(cand > r.m + kRescaleSlack) != 0) {
        const float corr = cand == -INFINITY ? 1.f : fast_exp2(r.m - cand);
        r.m = cand;
        r.l *= corr;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) r.o[t][i] *= corr;
    }
    const float shift = softmax_base(r.m);  // (no key yet: every s is -inf, and 2^-inf is 0)
    u32x4 p[2 * NT];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                e[i] = fast_exp2(fmaf(s[kt][8 * u + i], scale_log2, -shift));
                r.l += e[i];
            }
            p[2 * kt + u] = u32x4{pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]), pack_bf16x2(e[4], e[5]), pack_bf16x2(e[6], e[7])};
        }
    // A lane's keys of step `st`: 16 st + 4 half + 0..3 and 8 further, in the order that S^T leaves them.
    const int from = (lane & 15) >> 2;  // key of the four that the lane addresses
    const uint8_t* const base = reinterpret_cast<const uint8_t*>(lv);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int dim = 32 * t + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const uint8_t* const at = base + (from + 4 * half) * (2 * D) + 16 * v_chunk<D>(from, dim >> 3) + 8 * ((dim >> 2) & 1);
#pragma unroll
        for (int st = 0; st < 2 * NT; ++st) {
            const u32x2 v0 = lds_read_tr16(at + (16 * st) * (2 * D)), v1 = lds_read_tr16(at + (16 * st + 8) * (2 * D));
            const u32x4 v = {v0[0], v0[1], v1[0], v1[1]};
            if constexpr (UNEVEN) {
                bool odd = false;  // infinities or NaN
                if (mask) {
#pragma unroll
                    for (int w = 0; w < 4; ++w) odd = odd || (v[w] & 0x7F80u) == 0x7F80u || (v[w] & 0x7F800000u) == 0x7F800000u;
                }
                if (__ballot(odd) != 0) {
                    for (int k = 0; k < 16; ++k) {  // key k of the step alone; rows that do not see it keep what they have
                        const int in = (k & 3) + 4 * (k >> 3);  // its place among the 8 of its lanes
                        u32x4 one;
#pragma unroll
                        for (int w = 0; w < 4; ++w)
                            one[w] = half == ((k >> 2) & 1) && w == in >> 1 ? v[w] & (in & 1 ? 0xFFFF0000u : 0xFFFFu) : 0u;
                        const f32x16 sum = mfma32(one, p[st], r.o[t]);
                        const bool sees = key0 + 16 * st + k < r.limit;
#pragma unroll
                        for (int i = 0; i < 16; ++i) r.o[t][i] = sees ? sum[i] : r.o[t][i];
                    }
                    continue;
                }
            }
            r.o[t] = mfma32(v, p[st], r.o[t]);
        }
    }
}

// The lane's row of a partial: 4 dims a store, in the order of the registers.
template <int D>
__device__ __forceinline__ void store_partial(const PrefixArgs& a, const Rows<D>& r, float l, size_t row) {
    const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
            *reinterpret_cast<f32x4*>(a.part_o + row * D + 32 * t + 8 * i4 + 4 * half) =
                f32x4{r.o[t][4 * i4], r.o[t][4 * i4 + 1], r.o[t][4 * i4 + 2], r.o[t][4 * i4 + 3]};
    if (half == 0) reinterpret_cast<float2*>(a.part_ml)[row] = make_float2(r.m, l);
}

// ---- the prefix ---------------------------------------------------------------------------------------------

template <int D, bool E4M3, int TEAM>
__device__ __forceinline__ void prefix_task(const PrefixArgs& a, int index, uint8_t* lds, float2* lds_ml) {
    constexpr int NT = TEAM == 1 ? 1 : 2, KEYS = 32 * NT, TEAMS = kWaves / TEAM, NCH = D / 8;
    const int lane = threadIdx.x & 63, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile_of = wave % TEAM, team = wave / TEAM, t = threadIdx.x % (64 * TEAM);
    // kv heads in turn, so that consecutive work-groups (XCDs in turn) take one each and an L2 holds few heads' rows.
    const int h = index % a.cache.n_kv_heads, rest = index / a.cache.n_kv_heads;
    const int block = rest % a.blocks, piece = rest / a.blocks;
    const int begin = piece * a.chunk, end = min(begin + a.chunk, a.prefix_len);
    const int rows = a.batch * a.group, H_q = a.cache.n_kv_heads * a.group;

    const int row = (block * TEAM + tile_of) * 32 + col;
    const int b = row / a.group;
    Rows<D> r;
    rows_clear(r);
    r.limit = 0;
    if (row < rows) {
        r.limit = a.shared != nullptr ? min(a.shared[b], a.prefix_len) : a.prefix_len;
        const u32x4* const q = reinterpret_cast<const u32x4*>(a.q + ((size_t)b * H_q + h * a.group + (row - b * a.group)) * D);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) r.q[s] = q[2 * s + (lane >> 5)];
    } else {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) r.q[s] = u32x4{0u, 0u, 0u, 0u};
    }
    const int lo = __reduce_min_sync(~0ull, row < rows ? r.limit : INT_MAX);
    const int hi = __reduce_max_sync(~0ull, r.limit);

    u32x4* const lk = reinterpret_cast<u32x4*>(lds) + (size_t)team * 2 * KEYS * NCH;
    u32x4* const lv = lk + KEYS * NCH;
    const int tiles = (end - begin + KEYS - 1) / KEYS, rounds = (tiles + TEAMS - 1) / TEAMS;
    Staged<D, E4M3, NT, TEAM> staged;
    if (team < tiles) staged.load(a, a.prefix_b, h, begin + team * KEYS, end, t);
    for (int i = 0; i < rounds; ++i) {
        const int tile = i * TEAMS + team, key0 = begin + tile * KEYS;
        if (TEAM > 1 && i > 0) lds_barrier();  // the tile before is read
        if (tile < tiles) staged.store(lk, lv, t);
        if (tile + TEAMS < tiles) staged.load(a, a.prefix_b, h, key0 + TEAMS * KEYS, end, t);
        if constexpr (TEAM > 1) lds_barrier();
        else lds_done();
        if (tile < tiles && key0 < hi) attend<D, NT, true>(r, lk, lv, key0, lo, a.scale_log2);
    }
    // The teams meet in LDS: the others leave what they have, the first takes it.
    float l = pair_sum32(r.l);
    if constexpr (TEAMS > 1) {
        constexpr int WAVE_BYTES = 2 * KEYS * NCH * 16 / TEAM;  // of the tiles: 32 rows of O
        static_assert(WAVE_BYTES >= 32 * D * 4, "a wave's O takes its share of the tiles");
        f32x4* const lo4 = reinterpret_cast<f32x4*>(lds);
        lds_barrier();
        if (team > 0) {
#pragma unroll
            for (int m = 0; m < D / 32; ++m)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4)
                    lo4[((size_t)wave * (D / 8) + m * 4 + i4) * 64 + lane] =
                        f32x4{r.o[m][4 * i4], r.o[m][4 * i4 + 1], r.o[m][4 * i4 + 2], r.o[m][4 * i4 + 3]};
            if (lane < 32) lds_ml[wave * 32 + lane] = make_float2(r.m, l);
        }
        lds_barrier();
        if (team > 0) return;
        float M = r.m;
#pragma unroll
        for (int k = 1; k < TEAMS; ++k) M = fmaxf(M, lds_ml[(wave + k * TEAM) * 32 + col].x);
        const float base = softmax_base(M);
        const float mine = fast_exp2(r.m - base);
        l *= mine;
#pragma unroll
        for (int m = 0; m < D / 32; ++m)
#pragma unroll
            for (int i = 0; i < 16; ++i) r.o[m][i] *= mine;
#pragma unroll
        for (int k = 1; k < TEAMS; ++k) {
            const int other = wave + k * TEAM;
            const float2 ml = lds_ml[other * 32 + col];
            const float f = fast_exp2(ml.x - base);
            l = fmaf(f, ml.y, l);
#pragma unroll
            for (int m = 0; m < D / 32; ++m)
#pragma unroll
                for (int i4 = 0; i4 < 4; ++i4) {
                    const f32x4 v = lo4[((size_t)other * (D / 8) + m * 4 + i4) * 64 + lane];
#pragma unroll
                    for (int i = 0; i < 4; ++i) r.o[m][4 * i4 + i] = fmaf(f, v[i], r.o[m][4 * i4 + i]);
                }
        }
        r.m = M;
    }
    if (row < rows) store_partial<D>(a, r, l, ((size_t)piece * a.cache.n_kv_heads + h) * rows + row);
}

// ---- own rows -----------------------------------------------------------------------------------------------

// Appends the sequence's row (the call's k_new and v_new) to the cache: the wave's first lanes K, the next ones V.
template <int D, bool E4M3>
__device__ __forceinline__ void append_row(const PrefixArgs& a, int b, int h, int pos) {
    constexpr int LANES = D / 8;
    const int lane = threadIdx.x & 63;
    if (lane >= 2 * LANES) return;
    const int side = lane / LANES, at = lane % LANES;
    const u32x4 w = reinterpret_cast<const u32x4*>((side ? a.v_new : a.k_new) + ((size_t)b * a.cache.n_kv_heads + h) * D)[at];
    const int64_t row = kv8_row(a.cache, b, h, pos);
    uint8_t* const to = side ? a.cache.v : a.cache.k;
    if constexpr (E4M3) {
        float x[8];
        unpack_bf16x8(w, x);
        uint32_t byte;
        const u32x2 c = kv8_quantise<LANES>(x, &byte);
        if (row < 0) return;  // (unmapped: not written)
        reinterpret_cast<u32x2*>(to + row * D)[at] = c;
        if (at == 0) (side ? a.cache.v_scale : a.cache.k_scale)[row] = (uint8_t)byte;
    } else if (row >= 0) {
        reinterpret_cast<u32x4*>(to)[row * LANES + at] = w;
    }
}

// The same row as attention sees it, into row `key` of a tile in LDS.
template <int D, bool E4M3>
__device__ __forceinline__ void put_row(const PrefixArgs& a, int b, int h, int key, u32x4* lk, u32x4* lv) {
    constexpr int LANES = D / 8;
    const int lane = threadIdx.x & 63;
    if (lane >= 2 * LANES) return;
    const int side = lane / LANES, at = lane % LANES;
    u32x4 w = reinterpret_cast<const u32x4*>((side ? a.v_new : a.k_new) + ((size_t)b * a.cache.n_kv_heads + h) * D)[at];
    if constexpr (E4M3) {
        float x[8];
        unpack_bf16x8(w, x);
        uint32_t byte;
        const u32x2 c = kv8_quantise<LANES>(x, &byte);
        w = codes_to_bf16x8(c[0], c[1], kv8_scale(byte));
    }
    if (side) lv[key * LANES + v_chunk<D>(key, at)] = w;
    else lk[key * LANES + k_chunk<D>(key, at)] = w;
}

template <int D, bool E4M3>
__device__ __forceinline__ void own_tasks(const PrefixArgs& a, int index, uint8_t* lds, size_t part0) {
    constexpr int NCH = D / 8;
    const int lane = threadIdx.x & 63, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int H_q = a.cache.n_kv_heads * a.group, n_waves = a.own_wgs * kWaves, first = wave * a.own_wgs + index;
    u32x4* const lk = reinterpret_cast<u32x4*>(lds) + (size_t)wave * 2 * kOwnKeys * NCH;
    u32x4* const lv = lk + kOwnKeys * NCH;

    // The appended row of sequence b: inside the cache, and not among the prefix's rows, which others are reading.
    auto row_of = [&](int b) __attribute__((always_inline)) {
        if (a.k_new == nullptr) return -1;
        const int pos = a.positions[b];
        return pos < 0 || pos >= a.cache.l_max || (b == a.prefix_b && pos < a.prefix_len) ? -1 : pos;
    };
    if (a.k_new != nullptr)
        for (int u = first; u < a.batch * a.cache.n_kv_heads; u += n_waves) {
            const int b = u / a.cache.n_kv_heads, pos = row_of(b);
            if (pos >= 0) append_row<D, E4M3>(a, b, u - b * a.cache.n_kv_heads, pos);
        }

    const int log2 = own_log2(a);
    // Task i: kv head i % H_kv of piece i / H_kv, pieces of the sequences in order.
    int c0 = -64, before = 0, len = 0, upto = 0;  // a window of 64 sequences: pieces before it, a lane's own rows, its pieces' running sum
    int total = 0;
    for (int task = first;; task += n_waves) {
        const int piece = task / a.cache.n_kv_heads, h = task - piece * a.cache.n_kv_heads;
        while (piece >= total) {  // (tasks come in order: the window only moves on)
            c0 += 64;
            if (c0 >= a.batch) return;
            before = total;
            len = own_len(a, c0 + lane);
            upto = wave_scan(own_pieces(len, log2));
            total = before + __builtin_amdgcn_readlane(upto, 63);
        }
        const int at = (int)__builtin_ctzll(__ballot(before + upto > piece));
        const int L = __builtin_amdgcn_readlane(len, at), b = c0 + at;
        const int k = piece - before - (__builtin_amdgcn_readlane(upto, at) - own_pieces(L, log2));
        const int begin = k << log2, end = min((int64_t)L, ((int64_t)k + 1) << log2);
        const int pos = row_of(b);

        Rows<D> r;
        rows_clear(r);
        r.limit = L;
        Staged<D, E4M3, 1, 1> staged;
        staged.load(a, b, h, begin, end, lane);
        const u32x4* const q = reinterpret_cast<const u32x4*>(a.q + ((size_t)b * H_q + h * a.group + (col < a.group ? col : 0)) * D);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) r.q[s] = q[2 * s + (lane >> 5)];
        for (int key0 = begin; key0 < end; key0 += kOwnKeys) {
            asm volatile("" ::: "memory");  // (the tile before is read)
            staged.store(lk, lv, lane);
            if (key0 + kOwnKeys < end) staged.load(a, b, h, key0 + kOwnKeys, end, lane);
            if (pos >= key0 && pos < key0 + kOwnKeys && pos < end) {
                lds_done();
                put_row<D, E4M3>(a, b, h, pos - key0, lk, lv);
            }
            lds_done();
            attend<D, 1, false>(r, lk, lv, key0, end, a.scale_log2);
        }
        const float l = pair_sum32(r.l);
        if (col < a.group) store_partial<D>(a, r, l, part0 + (size_t)task * a.group + col);
    }
}

// ---- the launches --------------------------------------------------------------------------------------------

template <int D>
constexpr int tile_bytes() { return kWaves * 2 * kOwnKeys * D * 2; }

template <int D, bool E4M3, int TEAM>
__global__ __launch_bounds__(kWaves * 64, 2) void decode_prefix_kernel(PrefixArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[tile_bytes<D>()];
    __shared__ float2 lds_ml[kWaves * 32];
    // Work-groups in eights (one of each XCD): the prefix's and the others in turn while there are both.
    const int prefix_wgs = a.pieces * a.blocks * a.cache.n_kv_heads, own = a.own_wgs;
    const int block = wide_block(), eight = block >> 3, in = block & 7;
    const int both = min(prefix_wgs >> 3, own >> 3);
    int index;
    bool is_prefix;
    if (eight < 2 * both) {
        is_prefix = (eight & 1) == 0;
        index = (eight >> 1) * 8 + in;
    } else {
        index = block - 8 * both;  // (of what is left: the prefix's first)
        is_prefix = index < prefix_wgs;
        if (!is_prefix) index = block - prefix_wgs;
    }
    if (is_prefix) prefix_task<D, E4M3, TEAM>(a, index, lds, lds_ml);
    else if (index < own) own_tasks<D, E4M3>(a, index, lds, (size_t)a.pieces * a.cache.n_kv_heads * a.batch * a.group);
}

// Joins a query row's partials: a work-group per row, D / 4 threads for every (256 / (D / 4))-th of them.
constexpr int kMergeThreads = 256;
template <int D>
__global__ __launch_bounds__(kMergeThreads) void decode_prefix_merge_kernel(PrefixArgs a) {
    constexpr int E = D / 4, PARTS = kMergeThreads / E;
    const int block = wide_block(), H_q = a.cache.n_kv_heads * a.group, b = block / H_q, head = block - b * H_q;
    if (b >= a.batch) return;
    const int h = head / a.group, g = head - h * a.group, lane = threadIdx.x & 63;
    const int part = threadIdx.x / E, e = threadIdx.x % E;
    const int limit = a.shared != nullptr ? min(a.shared[b], a.prefix_len) : a.prefix_len;
    const int n_prefix = limit > 0 ? (limit + a.chunk - 1) / a.chunk : 0;
    const int log2 = own_log2(a);
    int before = 0;  // pieces of the sequences before this one
    for (int c0 = 0; c0 < b; c0 += 64)
        before += __builtin_amdgcn_readlane(wave_scan(c0 + lane < b ? own_pieces(own_len(a, c0 + lane), log2) : 0), 63);
    const int n_own = own_pieces(own_len(a, b), log2), n = n_prefix + n_own;
    const size_t rows = (size_t)a.batch * a.group;
    const size_t prefix_row = h * rows + (size_t)b * a.group + g, prefix_step = a.cache.n_kv_heads * rows;
    const size_t own_row = (size_t)a.pieces * prefix_step + ((size_t)before * a.cache.n_kv_heads + h) * a.group + g;
    const size_t own_step = (size_t)a.cache.n_kv_heads * a.group;
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int s = part; s < n; s += PARTS) {
        const size_t row = s < n_prefix ? prefix_row + s * prefix_step : own_row + (s - n_prefix) * own_step;
        const float2 ml = reinterpret_cast<const float2*>(a.part_ml)[row];
        const f32x4 o = reinterpret_cast<const f32x4*>(a.part_o + row * D)[e];
        const float m = fmaxf(M, ml.x), base = softmax_base(m);
        const float keep = fast_exp2(M - base), f = fast_exp2(ml.x - base);
        L = fmaf(f, ml.y, L * keep);
#pragma unroll
        for (int i = 0; i < 4; ++i) O[i] = fmaf(f, o[i], O[i] * keep);
        M = m;
    }
    __shared__ __attribute__((aligned(16))) float lds_o[PARTS * D];
    __shared__ float2 lds_ml[PARTS];
    reinterpret_cast<f32x4*>(lds_o)[part * E + e] = O;
    if (e == 0) lds_ml[part] = make_float2(M, L);
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += kMergeThreads) {
        float top = -INFINITY;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) top = fmaxf(top, lds_ml[p].x);
        const float base = softmax_base(top);
        float o = 0.f, l = 0.f;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const float f = fast_exp2(lds_ml[p].x - base);
            o = fmaf(f, lds_o[p * D + d], o);
            l = fmaf(f, lds_ml[p].y, l);
        }
        const size_t row = (size_t)b * H_q + head;
        a.out[row * D + d] = f32_to_bf16_rne(softmax_out(o, l));
        if (d == 0 && a.lse != nullptr) a.lse[row] = softmax_lse(top, l);
    }
}

template <int D, bool E4M3>
hipError_t launch_prefix_t(const PrefixArgs& a, const Launch& l) {
    const dim3 grid = wide_grid((int64_t)a.pieces * a.blocks * a.cache.n_kv_heads + a.own_wgs), block(kWaves * 64);
    if (a.row_tiles == 4) return launch_kernel(decode_prefix_kernel<D, E4M3, 4>, grid, block, l, a);
    if (a.row_tiles == 2) return launch_kernel(decode_prefix_kernel<D, E4M3, 2>, grid, block, l, a);
    return launch_kernel(decode_prefix_kernel<D, E4M3, 1>, grid, block, l, a);
}

}  // namespace

// Pieces of a prefix, whatever its length: with them the prefix's work-groups are about as many as CUs.
static int64_t most_pieces(const PrefixArgs& a, int n_cu) {
    return std::max<int64_t>(1, n_cu / ((int64_t)a.blocks * a.cache.n_kv_heads));
}

void plan_prefix(PrefixArgs* a, int n_cu) {
    const int64_t rows = (int64_t)a->batch * a->group;
    a->row_tiles = rows > 64 ? 4 : rows > 32 ? 2 : 1;
    a->blocks = (int)((rows + 32 * a->row_tiles - 1) / (32 * a->row_tiles));
    const int least = a->row_tiles == 1 ? 128 : 64 * (kWaves / a->row_tiles);  // keys of a round of a work-group
    const int64_t most = most_pieces(*a, n_cu), keys = (a->prefix_len + most - 1) / most;
    a->chunk = (int)std::max<int64_t>(least, (keys + least - 1) / least * least);
    a->pieces = a->prefix_len > 0 ? (int)(((int64_t)a->prefix_len + a->chunk - 1) / a->chunk) : 0;
    a->own_wgs = n_cu;
    a->own_slots = (int)std::max<int64_t>(kPrefixOwnSlots, (int64_t)a->batch * a->cache.n_kv_heads);
}

int64_t prefix_partial_rows_max(int batch, int n_kv_heads, int group, int n_cu) {
    PrefixArgs a{};
    a.batch = batch;
    a.group = group;
    a.cache.n_kv_heads = n_kv_heads;
    plan_prefix(&a, n_cu);
    return most_pieces(a, n_cu) * n_kv_heads * batch * group + (int64_t)a.own_slots * group;
}

hipError_t launch_decode_prefix(int head_dim, const PrefixArgs& a, const Launch& l) {
    const bool e4m3 = a.cache.k_scale != nullptr;
    if ((int64_t)a.pieces * a.blocks * a.cache.n_kv_heads + a.own_wgs > INT32_MAX) return hipErrorInvalidValue;
    if (head_dim == 128) return e4m3 ? launch_prefix_t<128, true>(a, l) : launch_prefix_t<128, false>(a, l);
    if (head_dim == 64) return e4m3 ? launch_prefix_t<64, true>(a, l) : launch_prefix_t<64, false>(a, l);
    return hipErrorInvalidValue;
}

hipError_t launch_decode_prefix_merge(int head_dim, const PrefixArgs& a, const Launch& l) {
    const int64_t wgs = (int64_t)a.batch * a.cache.n_kv_heads * a.group;
    if (wgs > INT32_MAX) return hipErrorInvalidValue;
    if (head_dim == 128) return launch_kernel(decode_prefix_merge_kernel<128>, wide_grid(wgs), dim3(kMergeThreads), l, a);
    if (head_dim == 64) return launch_kernel(decode_prefix_merge_kernel<64>, wide_grid(wgs), dim3(kMergeThreads), l, a);
    return hipErrorInvalidValue;
}

}  // namespace lara
