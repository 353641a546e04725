// Decode for a batch that shares a prefix: sequence b attends the first shared[b] rows of sequence prefix_b (which has none
// but its own) and then its own lens[b] rows, as one softmax,
//   o = sum over both of p_k v_k / sum of p_k,   p_k = exp(scale * q . k_k - m),
// and every row of the prefix is read for the whole batch, not once per sequence.
//
// The prefix's keys are cut into pieces and its query rows -- those of all sequences and of a kv head's group, [b][g] --
// into blocks of 32 * row_tiles; a work-group has a piece and a block.  Own rows are cut into pieces of a power of two keys,
// which the waves take when that is done.  All leave fp32 partials (O, m, l), which a second launch joins with log-sum-exp
// weights.
//
// One step, for 32 query rows and 32 or 64 keys, in both:
//   S^T [keys x 32 rows] = K . Q^T, O^T [D x 32 rows] += V^T . P^T by v_mfma_f32_32x32x16_bf16, with K and V in LDS (E4M3
// codes are turned to bf16, which holds them, on their way there) and one row's softmax in a lane pair.  Of the work-group's
// four waves row_tiles share a tile of K and V and the others take other tiles of the piece; a wave of own rows has its tile
// to itself.  The next tile's loads are under way while one is computed.
//
// p is rounded to bf16 before the second product (half a step, 2^-8 of it at most), l sums the unrounded ones; scores, sums
// and O are fp32.  A row is 0 (lse -inf) without keys, NaN with a score of NaN.  Rows of V that a sequence does not see do not
// reach it, whatever they hold: past the end they are read as zeros, and infinities and NaN of the prefix stay out of the
// products and are added to the rows that see them.
#include "decode_common.h"
#include "kv8_device.h"

#include <type_traits>

namespace lara {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef short i16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 8;
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

constexpr int kRoundKeys = 32 * kWaves;  // keys that a work-group has in LDS

// LDS of a work-group: K and V of 32 keys for each wave.
template <int D>
constexpr int tile_bytes() { return kWaves * 2 * kOwnKeys * D * 2; }

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

// A tile of NT * 32 keys on its way into LDS through the registers of TEAM waves; `t` is the thread's place among them.  ONCE:
// nothing else reads the rows (loads that pass the L2 stream faster).  FINITE: zeros take the place of infinities and NaN in V,
// and store() says whether there were any.
template <int D, bool E4M3, int NT, int TEAM, bool ONCE, bool FINITE>
struct Staged {
    static constexpr int NCH = D / 8, KEYS = 32 * NT, THREADS = 64 * TEAM;
    static constexpr int PIECES = E4M3 ? D / 16 : NCH;  // 16-byte loads of a row
    static constexpr int N = KEYS * PIECES / THREADS;
    static_assert(N >= 1 && N * THREADS == KEYS * PIECES, "whole loads");
    // Rows of up to 64 keys lie together (a page's, at least); a tile of more has two such parts.
    static constexpr int PARTS = KEYS > 64 ? KEYS / 64 : 1, PER = N / PARTS;
    static_assert(PARTS * PER == N, "loads of one part each");
    u32x4 k[N], v[N];
    uint8_t ks[N], vs[N];  // E4M3: scale bytes
    int live[PARTS];       // rows of a part that hold keys

    __device__ __forceinline__ void load(const PrefixArgs& a, int b, int h, int key0, int end, int t) {
        const uint32_t at = 16 * t, row_at = (uint32_t)t / PIECES;
#pragma unroll
        for (int g = 0; g < PARTS; ++g) {
            const int key = key0 + 64 * g < end ? key0 + 64 * g : key0;  // (a part behind the end: any rows that are there)
            int64_t row;
            if (a.cache.block_table == nullptr)
                row = ((int64_t)b * a.cache.n_kv_heads + h) * a.cache.l_cap + key;
            else
                row = paged_row_uniform(a.cache.block_table + (size_t)b * a.cache.max_pages, a.cache.page_shift, a.cache.n_kv_heads, h, key);
            live[g] = row < 0 ? 0 : end - key0 - 64 * g;  // (an unmapped page: rows of zeros, from any that is there)
            if (row < 0) row = 0;
            // (a uniform base and a 32-bit offset a lane)
            const uint8_t* const kp = a.cache.k + row * (PIECES * 16);
            const uint8_t* const vp = a.cache.v + row * (PIECES * 16);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const u32x4* const kfrom = reinterpret_cast<const u32x4*>(kp + i * (THREADS * 16) + at);
                const u32x4* const vfrom = reinterpret_cast<const u32x4*>(vp + i * (THREADS * 16) + at);
                k[g * PER + i] = ONCE ? __builtin_nontemporal_load(kfrom) : *kfrom;
                v[g * PER + i] = ONCE ? __builtin_nontemporal_load(vfrom) : *vfrom;
            }
            if constexpr (E4M3)
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    ks[g * PER + i] = (a.cache.k_scale + row + i * (THREADS / PIECES))[row_at];
                    vs[g * PER + i] = (a.cache.v_scale + row + i * (THREADS / PIECES))[row_at];
                }
        }
    }
    __device__ __forceinline__ bool store(u32x4* lk, u32x4* lv, int t) {
        bool odd = false;
        if constexpr (FINITE) odd = clear_odd();
        auto put = [&](int part, int key, int c, u32x4 kw, u32x4 vw) __attribute__((always_inline)) {
            if (live[part] < (KEYS < 64 ? KEYS : 64) && key - 64 * part >= live[part]) kw = vw = u32x4{0u, 0u, 0u, 0u};
            lk[key * NCH + k_chunk<D>(key, c)] = kw;
            lv[key * NCH + v_chunk<D>(key, c)] = vw;
        };
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int slot = i * THREADS + t, key = slot / PIECES, c = slot % PIECES;
            if constexpr (E4M3) {
                const float kscale = kv8_scale(ks[i]), vscale = kv8_scale(vs[i]);
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    put(i / PER, key, 2 * c + half, codes_to_bf16x8(k[i][2 * half], k[i][2 * half + 1], kscale),
                        codes_to_bf16x8(v[i][2 * half], v[i][2 * half + 1], vscale));
            } else {
                put(i / PER, key, c, k[i], v[i]);
            }
        }
        return odd;
    }

  private:
    // Zeros for infinities and NaN among the V values in the registers; whether there were any (in rows behind the end, too:
    // add_odd() looks closer).  A value's exponent of ones (a code's seven ones) carries into the bit above it.
    __device__ __forceinline__ bool clear_odd() {
        constexpr uint32_t FIELD = E4M3 ? 0x7F7F7F7Fu : 0x7F807F80u, ONE = E4M3 ? 0x01010101u : 0x00800080u, TOP = E4M3 ? 0x80808080u : 0x80008000u;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) any |= (v[i][j] & FIELD) + ONE;
        if (__ballot((any & TOP) != 0) == 0) return false;
        constexpr int BITS = E4M3 ? 8 : 16;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t at = (((v[i][j] & FIELD) + ONE) & TOP) >> (BITS - 1);  // a one for each
                v[i][j] &= ~(at * ((1u << BITS) - 1u));
            }
        return (any & TOP) != 0;
    }
};

// The tile of keys key0 .. in LDS, for 32 rows.
template <int D, int NT>
__device__ __forceinline__ void attend(Rows<D>& r, const u32x4* lk, const u32x4* lv, int key0, float scale_log2) {
    constexpr int NCH = D / 8, STEPS = D / 16, MT = D / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    f32x16 s[NT];
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kt][i] = 0.f;
    // Fragments are read a few steps before their products, and no further (sched_barrier): registers would not hold them.
    constexpr int kAhead = 2;
    u32x4 kf[STEPS][NT];
    auto read_k = [&](int st) __attribute__((always_inline)) {
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) kf[st][kt] = lk[(32 * kt + col) * NCH + k_chunk<D>(col, 2 * st + half)];
    };
#pragma unroll
    for (int st = 0; st < kAhead; ++st) read_k(st);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
        if (st + kAhead < STEPS) read_k(st + kAhead);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kt = 0; kt < NT; ++kt) s[kt] = mfma32(kf[st][kt], r.q[st], s[kt]);
    }
    // Keys that a row does not see (every tile: a branch around it costs more, in copies of O that registers do not hold).
    float mx = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < NT; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[kt][i] = 32 * kt + 8 * (i >> 2) + (i & 3) < r.limit - key0 - 4 * half ? s[kt][i] : -INFINITY;
            mx = fmaxf(mx, s[kt][i]);
        }
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
    const float shift = softmax_base(r.m);  // (no key yet: every score is -inf, and 2^-inf is 0)
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
    auto value = [&](int t, int st) __attribute__((always_inline)) {
        const int dim = 32 * t + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const uint8_t* const at = base + (from + 4 * half + 16 * st) * (2 * D) + 16 * v_chunk<D>(from, dim >> 3) + 8 * ((dim >> 2) & 1);
        const u32x2 v0 = lds_read_tr16(at), v1 = lds_read_tr16(at + 8 * (2 * D));
        return u32x4{v0[0], v0[1], v1[0], v1[1]};
    };
    constexpr int PV = MT * 2 * NT, kAheadV = 3;
    u32x4 vf[PV];
#pragma unroll
    for (int i = 0; i < kAheadV; ++i) vf[i] = value(i / (2 * NT), i % (2 * NT));
#pragma unroll
    for (int i = 0; i < PV; ++i) {
        if (i + kAheadV < PV) vf[i + kAheadV] = value((i + kAheadV) / (2 * NT), (i + kAheadV) % (2 * NT));
        __builtin_amdgcn_sched_barrier(0);
        r.o[i / (2 * NT)] = mfma32(vf[i], p[i % (2 * NT)], r.o[i / (2 * NT)]);
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

// Query rows that attend it, per kv head: every sequence's but its own.
__host__ __device__ inline int prefix_rows(const PrefixArgs& a) { return (a.batch - 1) * a.group; }

// Adds the infinities and NaN among the V rows of a run's keys begin + from .., begin + from + step .., `n` each, to the rows
// that see them.  (Rare, and slow: values come one by one from the cache.)
template <int D, bool E4M3>
__device__ __forceinline__ float odd_value(const PrefixArgs& a, int h, int key, int dim) {
    const int64_t row = kv8_row(a.cache, a.prefix_b, h, key);
    if (row < 0) return 0.f;
    float v;
    if constexpr (E4M3) {
        const uint32_t code = a.cache.v[row * D + dim];
        v = (code & 0x7Fu) == 0x7Fu ? __uint_as_float(0x7FC00000u) : 0.f;
    } else {
        v = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(a.cache.v)[row * D + dim] << 16);
    }
    return fabsf(v) < INFINITY ? 0.f : v;
}
template <int D, bool E4M3>
__device__ __forceinline__ void add_odd(Rows<D>& r, const PrefixArgs& a, int h, int begin, int end, int from, int step, int n) {
    const int half = (threadIdx.x & 63) >> 5;
    for (int k0 = begin + from; k0 < end; k0 += step)
        for (int key = k0; key < min(k0 + n, end); ++key)
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float v = odd_value<D, E4M3>(a, h, key, 32 * t + 8 * (i >> 2) + 4 * half + (i & 3));
                    if (key < r.limit) r.o[t][i] += v;
                }
}

// TEAM waves share 32 * TEAM keys in LDS at a time, for 32 rows each; the work-group's TEAMS teams take the others of a round.
template <int D, bool E4M3, int TEAM>
__device__ __forceinline__ void prefix_task(const PrefixArgs& a, int index, uint8_t* lds, float2* lds_ml, int* lds_odd) {
    constexpr int NT = 1, KEYS = 32 * TEAM, TEAMS = kWaves / TEAM, NCH = D / 8;
    const int lane = threadIdx.x & 63, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile_of = wave % TEAM, team = wave / TEAM, t = threadIdx.x % (64 * TEAM);
    // kv heads in turn, so that consecutive work-groups (XCDs in turn) take one each and an L2 holds few heads' rows.
    const int h = index % a.cache.n_kv_heads, rest = index / a.cache.n_kv_heads;
    const int block = rest % a.blocks, piece = rest / a.blocks;
    const int begin = piece * a.chunk, end = min(begin + a.chunk, a.prefix_len);
    const int rows = prefix_rows(a), H_q = a.cache.n_kv_heads * a.group;

    u32x4* const lk = reinterpret_cast<u32x4*>(lds) + (size_t)team * 2 * KEYS * NCH;
    u32x4* const lv = lk + KEYS * NCH;
    Staged<D, E4M3, TEAM, TEAM, false, true> staged;
    if (begin + team * KEYS < end) staged.load(a, a.prefix_b, h, begin + team * KEYS, end, t);

    const int row = (block * TEAM + tile_of) * 32 + col;
    int b = row / a.group;
    const int g = row - b * a.group;
    if (b >= a.prefix_b) ++b;
    Rows<D> r;
    rows_clear(r);
    r.limit = 0;
    if (row < rows) {
        r.limit = a.shared != nullptr ? min(a.shared[b], a.prefix_len) : a.prefix_len;
        const u32x4* const q = reinterpret_cast<const u32x4*>(a.q + ((size_t)b * H_q + h * a.group + g) * D);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) r.q[s] = q[2 * s + (lane >> 5)];
    } else {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) r.q[s] = u32x4{0u, 0u, 0u, 0u};
    }
    const int hi = min(__reduce_max_sync(~0ull, r.limit), end);

    // (lds_odd[wave]: some V of the wave's keys was not finite; each wave writes its own and reads its team's behind a barrier)
    bool odd = false;
    for (int round = begin; round < end; round += kRoundKeys) {
        const int key0 = round + team * KEYS;
        if (TEAM > 1 && round > begin) lds_barrier();  // the round before is read
        if (key0 < end) odd |= staged.store(lk, lv, t);
        if (key0 + kRoundKeys < end) staged.load(a, a.prefix_b, h, key0 + kRoundKeys, end, t);
        if constexpr (TEAM > 1) lds_barrier();
        else lds_done();
        for (int k = 0; k < KEYS; k += 32 * NT)
            if (key0 + k < hi) attend<D, NT>(r, lk + k * NCH, lv + k * NCH, key0 + k, a.scale_log2);
    }
    // What is not finite reaches the rows that see it, and no others: 0 times it would be NaN in the products.
    odd = __ballot(odd) != 0;
    if (lane == 0) lds_odd[wave] = odd;
    lds_barrier();
#pragma unroll
    for (int w = 0; w < TEAM; ++w) odd = odd || lds_odd[team * TEAM + w] != 0;
    if (odd) add_odd<D, E4M3>(r, a, h, begin, end, team * KEYS, kRoundKeys, KEYS);
    // The teams meet in LDS, every wave's O row by row (16-byte words permuted by the row: no bank is met twice), and leave it
    // as whole rows.
    constexpr int WORDS = D / 4;
    f32x4* const lo = reinterpret_cast<f32x4*>(lds);
    const float l = pair_sum32(r.l);
    lds_barrier();  // (the tiles are read)
#pragma unroll
    for (int m = 0; m < D / 32; ++m)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
            lo[(wave * 32 + col) * WORDS + ((8 * m + 2 * i4 + (lane >> 5)) ^ (col & (WORDS - 1)))] =
                f32x4{r.o[m][4 * i4], r.o[m][4 * i4 + 1], r.o[m][4 * i4 + 2], r.o[m][4 * i4 + 3]};
    if (lane < 32) lds_ml[wave * 32 + lane] = make_float2(r.m, l);
    lds_barrier();
    const int row0 = block * TEAM * 32;
    const size_t to = ((size_t)piece * a.cache.n_kv_heads + h) * rows + row0;
    for (int i = threadIdx.x; i < TEAM * 32 * WORDS; i += kWaves * 64) {
        const int at = i / WORDS, word = i % WORDS;  // row of the block
        if (row0 + at >= rows) break;
        float M = lds_ml[at].x;
#pragma unroll
        for (int k = 1; k < TEAMS; ++k) M = fmaxf(M, lds_ml[k * TEAM * 32 + at].x);
        const float base = softmax_base(M);
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
        float L = 0.f;
#pragma unroll
        for (int k = 0; k < TEAMS; ++k) {
            const int from = k * TEAM * 32 + at;
            const float2 ml = lds_ml[from];
            const float f = fast_exp2(ml.x - base);
            const f32x4 v = lo[from * WORDS + (word ^ (at & 31 & (WORDS - 1)))];
            L = fmaf(f, ml.y, L);
#pragma unroll
            for (int j = 0; j < 4; ++j) O[j] = fmaf(f, v[j], O[j]);
        }
        reinterpret_cast<f32x4*>(a.part_o)[(to + at) * WORDS + word] = O;
        if (word == 0) reinterpret_cast<float2*>(a.part_ml)[to + at] = make_float2(M, L);
    }
    lds_barrier();  // (own rows follow in the same LDS)
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
__device__ __forceinline__ void own_tasks(const PrefixArgs& a, int index, int prefix_wgs, int wgs, uint8_t* lds, size_t part0) {
    constexpr int NCH = D / 8;
    const int lane = threadIdx.x & 63, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int H_q = a.cache.n_kv_heads * a.group;
    const int n_waves = wgs * kWaves, me = wave * wgs + index;
    u32x4* const lk = reinterpret_cast<u32x4*>(lds) + (size_t)wave * 2 * kOwnKeys * NCH;
    u32x4* const lv = lk + kOwnKeys * NCH;

    // The appended row of sequence b: inside the cache, and not among the prefix's rows, which others are reading.
    auto row_of = [&](int b) __attribute__((always_inline)) {
        if (a.k_new == nullptr) return -1;
        const int pos = a.positions[b];
        return pos < 0 || pos >= a.cache.l_max || (b == a.prefix_b && pos < a.prefix_len) ? -1 : pos;
    };
    if (a.k_new != nullptr)
        for (int u = me; u < a.batch * a.cache.n_kv_heads; u += n_waves) {
            const int b = u / a.cache.n_kv_heads, pos = row_of(b);
            if (pos >= 0) append_row<D, E4M3>(a, b, u - b * a.cache.n_kv_heads, pos);
        }

    const int log2 = own_log2(a);
    // Tasks are dealt to the waves in turn.  Those of work-groups that had a part of the prefix come late: the others get the
    // first `ahead` rounds alone (a round of the prefix, 256 keys, takes about as long as 32 own keys on every wave, and its
    // beginning and end as two more).
    const int others = (wgs - prefix_wgs) * kWaves, late = 2 + a.chunk / kRoundKeys;
    const int ahead = others > 0 && prefix_wgs > 0 ? max(1, late * kOwnKeys >> log2) : 0;
    const bool is_late = index < prefix_wgs;
    const int me_first = is_late ? 0 : wave * (wgs - prefix_wgs) + index - prefix_wgs;
    auto task_at = [&](int n) __attribute__((always_inline)) {  // the wave's n-th
        if (is_late || n >= ahead) return ahead * others + (n - (is_late ? 0 : ahead)) * n_waves + me;
        return n * others + me_first;
    };
    // Task i: kv head i % H_kv of piece i / H_kv, pieces of the sequences in order; a step is 32 keys of one.  What is loaded
    // is a step ahead of what is computed, across tasks.
    struct Step {
        int task, b, h, L, key, end;
    };
    int c0 = -64, before = 0, len = 0, upto = 0;  // a window of 64 sequences: pieces before it, a lane's own rows, its pieces' running sum
    int total = 0;
    auto open = [&](Step& s) __attribute__((always_inline)) -> bool {
        const int piece = s.task / a.cache.n_kv_heads;
        while (piece >= total) {  // (tasks come in order: the window only moves on)
            c0 += 64;
            if (c0 >= a.batch) return false;
            before = total;
            len = own_len(a, c0 + lane);
            upto = wave_scan(own_pieces(len, log2));
            total = before + __builtin_amdgcn_readlane(upto, 63);
        }
        const int at = (int)__builtin_ctzll(__ballot(before + upto > piece));
        s.L = __builtin_amdgcn_readlane(len, at);
        s.b = c0 + at;
        s.h = s.task - piece * a.cache.n_kv_heads;
        const int k = piece - before - (__builtin_amdgcn_readlane(upto, at) - own_pieces(s.L, log2));
        s.key = k << log2;
        s.end = (int)min((int64_t)s.L, ((int64_t)k + 1) << log2);
        return true;
    };
    Step now, next;
    int n = 0;
    now.task = task_at(0);
    if (!open(now)) return;
    next = now;
    Staged<D, E4M3, 1, 1, true, false> staged;
    staged.load(a, now.b, now.h, now.key, now.end, lane);
    Rows<D> r;
    int pos = -1;
    bool opening = true, more = true;
    do {
        if (opening) {
            rows_clear(r);
            r.limit = now.L;
            const u32x4* const q = reinterpret_cast<const u32x4*>(a.q + ((size_t)now.b * H_q + now.h * a.group + (col < a.group ? col : 0)) * D);
#pragma unroll
            for (int s = 0; s < D / 16; ++s) r.q[s] = q[2 * s + (lane >> 5)];
            pos = row_of(now.b);
        }
        next.key += kOwnKeys;
        const bool closing = next.key >= next.end;
        if (closing) {
            next.task = task_at(++n);
            more = open(next);
        }
        asm volatile("" ::: "memory");  // (the tile before is read)
        staged.store(lk, lv, lane);
        if (more) staged.load(a, next.b, next.h, next.key, next.end, lane);
        if (pos >= now.key && pos < now.key + kOwnKeys && pos < now.end) {
            lds_done();
            put_row<D, E4M3>(a, now.b, now.h, pos - now.key, lk, lv);
        }
        lds_done();
        attend<D, 1>(r, lk, lv, now.key, a.scale_log2);
        if (closing) {
            const float l = pair_sum32(r.l);
            if (col < a.group) store_partial<D>(a, r, l, part0 + (size_t)now.task * a.group + col);
        }
        now = next;
        opening = closing;
    } while (more);
}

// ---- the launches --------------------------------------------------------------------------------------------

template <int D, bool E4M3, int TEAM>
__global__ __launch_bounds__(kWaves * 64, 2) void decode_prefix_kernel(PrefixArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[tile_bytes<D>()];
    __shared__ float2 lds_ml[kWaves * 32];
    __shared__ int lds_odd[kWaves];
    // A work-group has a part of the prefix, if there are so many, and then some of the own rows.
    const int prefix_wgs = a.pieces * a.blocks * a.cache.n_kv_heads, wgs = max(prefix_wgs, a.own_wgs), index = wide_block();
    if (index >= wgs) return;
    if (index < prefix_wgs) prefix_task<D, E4M3, TEAM>(a, index, lds, lds_ml, lds_odd);
    own_tasks<D, E4M3>(a, index, prefix_wgs, wgs, lds, (size_t)a.pieces * a.cache.n_kv_heads * prefix_rows(a));
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
    const int limit = b == a.prefix_b ? 0 : a.shared != nullptr ? min(a.shared[b], a.prefix_len) : a.prefix_len;
    const int n_prefix = limit > 0 ? (limit + a.chunk - 1) / a.chunk : 0;
    const int log2 = own_log2(a);
    int before = 0;  // pieces of the sequences before this one
    for (int c0 = 0; c0 < b; c0 += 64)
        before += __builtin_amdgcn_readlane(wave_scan(c0 + lane < b ? own_pieces(own_len(a, c0 + lane), log2) : 0), 63);
    const int n_own = own_pieces(own_len(a, b), log2), n = n_prefix + n_own;
    const size_t rows = prefix_rows(a);
    const size_t prefix_row = h * rows + (size_t)(b - (b > a.prefix_b ? 1 : 0)) * a.group + g, prefix_step = a.cache.n_kv_heads * rows;
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
    const dim3 grid = wide_grid(std::max<int64_t>((int64_t)a.pieces * a.blocks * a.cache.n_kv_heads, a.own_wgs)), block(kWaves * 64);
    if (a.row_tiles == 4) return launch_kernel(decode_prefix_kernel<D, E4M3, 4>, grid, block, l, a);
    if (a.row_tiles == 2) return launch_kernel(decode_prefix_kernel<D, E4M3, 2>, grid, block, l, a);
    return launch_kernel(decode_prefix_kernel<D, E4M3, 1>, grid, block, l, a);
}

}  // namespace

// Pieces of a prefix, whatever its length: with them the prefix's work-groups are about as many as CUs.
static int64_t most_pieces(const PrefixArgs& a, int n_cu) {
    return std::max<int64_t>(1, n_cu / std::max<int64_t>(1, (int64_t)a.blocks * a.cache.n_kv_heads));
}

void plan_prefix(PrefixArgs* a, int n_cu) {
    const int64_t rows = prefix_rows(*a);
    a->row_tiles = rows > 64 ? 4 : rows > 32 ? 2 : 1;
    a->blocks = (int)((rows + 32 * a->row_tiles - 1) / (32 * a->row_tiles));
    const int least = kRoundKeys;
    const int64_t most = most_pieces(*a, n_cu), keys = (a->prefix_len + most - 1) / most;
    a->chunk = (int)std::max<int64_t>(least, (keys + least - 1) / least * least);
    a->pieces = a->prefix_len > 0 && rows > 0 ? (int)(((int64_t)a->prefix_len + a->chunk - 1) / a->chunk) : 0;
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
    if ((int64_t)a.pieces * a.blocks * a.cache.n_kv_heads > INT32_MAX / kWaves) return hipErrorInvalidValue;
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
