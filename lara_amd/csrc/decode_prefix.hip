// Decode for a batch that shares a prefix: sequence b attends the first shared[b] rows of sequence prefix_b (which has none
// but its own) and then its own lens[b] rows, as one softmax,
//   o = sum over both of p_k v_k / sum of p_k,   p_k = exp(scale * q . k_k - m),
// and every row of the prefix is read for the whole batch, not once per sequence.
//
// The prefix's keys are cut into pieces and its query rows -- those of all sequences and of a kv head's group, [b][g] --
// into blocks of 32 * row_tiles; a work-group has a piece and a block.  Own rows are cut into pieces of a power of two keys,
// which the waves take when that is done.  All leave fp32 partials (O, m, l), which a second launch joins with log-sum-exp
// weights.  Short contexts of few sequences take one launch without partials instead (decode_prefix_whole_kernel).
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
//
// 32 query heads over 8 of 128, us beside other launches (alone, both launches): 64 sequences behind 4096 rows with up to
// 256 of their own 18.2 (21 + 7.5), of which 7.4 are their own rows (35 MB), 3.6 the products and 6.7 staging, partials (17
// MB) and latency; 24 sequences of 64 heads behind 16384 29 (46 + 7.7), bound by a wave's chain of scores, maximum,
// exponentials and V.  Two work-groups of four waves a CU: with eight waves over 256 keys and one work-group 27.3 and 37.9.
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
constexpr int kOwnKeys = kPrefixOwnKeys;

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
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

// The same for transposing reads of eight (own rows).
template <int D>
__device__ __forceinline__ int v_chunk_own(int row, int c) {
    return c ^ 2 * (D == 128 ? row & 7 : (row >> 1) & 3);
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
constexpr int kWholeWaves = 8, kWholeValues = 1024 * 128;  // the most K values of a (sequence, kv head) for one work-group

// LDS of a work-group: K and V of 32 keys for each wave.
template <int D>
constexpr int tile_bytes() { return kWaves * 2 * kOwnKeys * D * 2; }

// ---- runs of own rows ------------------------------------------------------------------------------------

__device__ __forceinline__ int own_len(const PrefixArgs& a, int s) { return s < a.batch ? clamp_len(a.lens[s], a.cache.l_max) : 0; }
__device__ __forceinline__ int own_steps(int len) { return (len + kOwnKeys - 1) / kOwnKeys; }

// The steps (32 keys) of all (sequence, kv head)s in order are cut into one run for every wave of the launch: `first` steps
// for the first `others` waves and `rest` for the others, those of work-groups that had a part of the prefix and come late
// by about as many steps as the difference.  It follows from the lengths, so that both launches know it (all steps are at
// most 2^30: the caller sees to it).  A part of a (sequence, kv head) u in the run of wave w leaves its partial in slot u + w
// (one of the two rises from part to part).
struct Runs {
    int others, first, rest;
    int before;  // steps of a kv head's sequences before `b`
    __device__ __forceinline__ Runs(const PrefixArgs& a, int prefix_wgs, int wgs, int b) {
        const int lane = threadIdx.x & 63;
        int steps = 0;
        before = 0;
        for (int c0 = 0; c0 < a.batch; c0 += 64) {
            const int of = own_steps(own_len(a, c0 + lane)), upto = wave_scan(of);
            if (b >= c0 && b < c0 + 64) before = steps + __builtin_amdgcn_readlane(upto - of, b - c0);
            steps += __builtin_amdgcn_readlane(upto, 63);
        }
        steps *= a.cache.n_kv_heads;
        others = (wgs - prefix_wgs) * kWaves;
        const int waves = wgs * kWaves;
        const int late = others > 0 && prefix_wgs > 0 ? kLateSteps + a.chunk / kRoundKeys : 0;
        rest = steps > others * late ? (steps - others * late + waves - 1) / waves : 0;
        first = rest > 0 ? rest + late : others > 0 ? (steps + others - 1) / others : 0;
    }
    // Where wave w's run begins, and the wave in whose run step `at` lies.
    __device__ __forceinline__ int begin(int w) const { return w < others ? w * first : others * first + (w - others) * rest; }
    __device__ __forceinline__ int wave_of(int at) const { return at < others * first ? at / first : others + (at - others * first) / rest; }
    static constexpr int kLateSteps = 6;  // a part of the prefix costs about this and a step for each of its rounds
};

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

// A wave's share of a tile on its way into LDS: 32 keys for each wave that the tile serves.
template <int D, bool E4M3>
struct Loaded {
    static constexpr int PIECES = E4M3 ? D / 16 : D / 8;  // 16-byte loads of a row
    static constexpr int N = 32 * PIECES / 64;
    u32x4 k[N], v[N];
    uint8_t ks[N], vs[N];  // E4M3: scale bytes
    int live[2];           // rows that hold keys, of the first 64 and the others
};

// A tile of 32 * TEAM keys, loaded by TEAM waves; `t` is the thread's place among them.  OWN: nothing else reads the rows
// (loads that pass the L2 stream faster); the others' V has zeros for infinities and NaN, and store() says whether there were
// any.
template <int D, bool E4M3, int TEAM, bool OWN>
struct Staged {
    using Share = Loaded<D, E4M3>;
    static constexpr int NCH = D / 8, KEYS = 32 * TEAM, THREADS = 64 * TEAM;
    static constexpr int PIECES = Loaded<D, E4M3>::PIECES, N = Loaded<D, E4M3>::N;
    // Rows of up to 64 keys lie together (a page's, at least); a tile of more has two such parts.
    static constexpr int PARTS = KEYS > 64 ? KEYS / 64 : 1, PER = N / PARTS;
    static_assert(PARTS * PER == N, "loads of one part each");
    static_assert(PARTS <= 2, "live");

    __device__ static __forceinline__ void load(Share& x, const PrefixArgs& a, int b, int h, int key0, int end, int t) {
        const uint32_t at = 16 * t, row_at = (uint32_t)t / PIECES;
#pragma unroll
        for (int g = 0; g < PARTS; ++g) {
            const int key = key0 + 64 * g < end ? key0 + 64 * g : key0;  // (a part behind the end: any rows that are there)
            int64_t row;
            if (a.cache.block_table == nullptr)
                row = ((int64_t)b * a.cache.n_kv_heads + h) * a.cache.l_cap + key;
            else
                row = paged_row_uniform(a.cache.block_table + (size_t)b * a.cache.max_pages, a.cache.page_shift, a.cache.n_kv_heads, h, key);
            x.live[g] = row < 0 ? 0 : end - key0 - 64 * g;  // (an unmapped page: rows of zeros, from any that is there)
            if (row < 0) row = 0;
            // (a uniform base and a 32-bit offset a lane)
            const uint8_t* const kp = a.cache.k + row * (PIECES * 16);
            const uint8_t* const vp = a.cache.v + row * (PIECES * 16);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const u32x4* const kfrom = reinterpret_cast<const u32x4*>(kp + i * (THREADS * 16) + at);
                const u32x4* const vfrom = reinterpret_cast<const u32x4*>(vp + i * (THREADS * 16) + at);
                x.k[g * PER + i] = OWN ? __builtin_nontemporal_load(kfrom) : *kfrom;
                x.v[g * PER + i] = OWN ? __builtin_nontemporal_load(vfrom) : *vfrom;
            }
            if constexpr (E4M3)
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    x.ks[g * PER + i] = (a.cache.k_scale + row + i * (THREADS / PIECES))[row_at];
                    x.vs[g * PER + i] = (a.cache.v_scale + row + i * (THREADS / PIECES))[row_at];
                }
        }
    }
    __device__ static __forceinline__ bool store(Share& x, u32x4* lk, u32x4* lv, int t) {
        bool odd = false;
        if constexpr (!OWN) odd = clear_odd(x);
        auto put = [&](int part, int key, int c, u32x4 kw, u32x4 vw) __attribute__((always_inline)) {
            if (x.live[part] < (KEYS < 64 ? KEYS : 64) && key - 64 * part >= x.live[part]) kw = vw = u32x4{0u, 0u, 0u, 0u};
            lk[key * NCH + k_chunk<D>(key, c)] = kw;
            lv[key * NCH + (OWN ? v_chunk_own<D>(key, c) : v_chunk<D>(key, c))] = vw;
        };
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int slot = i * THREADS + t, key = slot / PIECES, c = slot % PIECES;
            if constexpr (E4M3) {
                const float kscale = kv8_scale(x.ks[i]), vscale = kv8_scale(x.vs[i]);
#pragma unroll
                for (int half = 0; half < 2; ++half)
                    put(i / PER, key, 2 * c + half, codes_to_bf16x8(x.k[i][2 * half], x.k[i][2 * half + 1], kscale),
                        codes_to_bf16x8(x.v[i][2 * half], x.v[i][2 * half + 1], vscale));
            } else {
                put(i / PER, key, c, x.k[i], x.v[i]);
            }
        }
        return odd;
    }

  private:
    // Zeros for infinities and NaN among the V values in the registers; whether there were any (in rows behind the end, too:
    // add_odd() looks closer).  A value's exponent of ones (a code's seven ones) carries into the bit above it.
    __device__ static __forceinline__ bool clear_odd(Share& x) {
        constexpr uint32_t FIELD = E4M3 ? 0x7F7F7F7Fu : 0x7F807F80u, ONE = E4M3 ? 0x01010101u : 0x00800080u, TOP = E4M3 ? 0x80808080u : 0x80008000u;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) any |= (x.v[i][j] & FIELD) + ONE;
        if (__ballot((any & TOP) != 0) == 0) return false;
        constexpr int BITS = E4M3 ? 8 : 16;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t at = (((x.v[i][j] & FIELD) + ONE) & TOP) >> (BITS - 1);  // a one for each
                x.v[i][j] &= ~(at * ((1u << BITS) - 1u));
            }
        return (any & TOP) != 0;
    }
};

// 32 keys from key0 on, in LDS, for 32 rows.
template <int D>
__device__ __forceinline__ void attend(Rows<D>& r, const u32x4* lk, const u32x4* lv, int key0, float scale_log2) {
    constexpr int NCH = D / 8, STEPS = D / 16, MT = D / 32;
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
    f32x16 s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) s = mfma32(lk[col * NCH + k_chunk<D>(col, 2 * st + half)], r.q[st], s);
    // Keys that a row does not see (in every tile: a branch around it costs more, in copies of O that registers do not hold).
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        s[i] = 8 * (i >> 2) + (i & 3) < r.limit - key0 - 4 * half ? s[i] : -INFINITY;
        mx = fmaxf(mx, s[i]);
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
    u32x4 p[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            e[i] = fast_exp2(fmaf(s[8 * u + i], scale_log2, -shift));
            r.l += e[i];
        }
        p[u] = u32x4{pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]), pack_bf16x2(e[4], e[5]), pack_bf16x2(e[6], e[7])};
    }
    // A lane's keys of step `st`: 16 st + 4 half + 0..3 and 8 further, in the order that S^T leaves them.
    const int from = (lane & 15) >> 2;  // key of the four that the lane addresses
    const uint8_t* const base = reinterpret_cast<const uint8_t*>(lv);
    auto value = [&](int i) __attribute__((always_inline)) {  // tile i / 2, step i % 2
        const int dim = 32 * (i / 2) + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        const uint8_t* const at = base + (from + 4 * half + 16 * (i % 2)) * (2 * D) + 16 * v_chunk<D>(from, dim >> 3) + 8 * ((dim >> 2) & 1);
        const u32x2 v0 = lds_read_tr16(at), v1 = lds_read_tr16(at + 8 * (2 * D));
        return u32x4{v0[0], v0[1], v1[0], v1[1]};
    };
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) r.o[i / 2] = mfma32(value(i), p[i % 2], r.o[i / 2]);
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

// last() is called when the last rows are in LDS: what it loads into `first` comes while they are worked on.
// TEAM waves share 32 * TEAM keys in LDS at a time, for 32 rows each; the work-group's TEAMS teams take the others of a round.
template <int D, bool E4M3, int TEAM, typename Last>
__device__ __forceinline__ void prefix_task(const PrefixArgs& a, int index, uint8_t* lds, float2* lds_ml, int* lds_odd, Loaded<D, E4M3>& first, Last&& last) {
    constexpr int KEYS = 32 * TEAM, TEAMS = kWaves / TEAM, NCH = D / 8;
    const int lane = threadIdx.x & 63, col = lane & 31, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tile_of = wave % TEAM, team = wave / TEAM, t = threadIdx.x % (64 * TEAM);
    // kv heads in turn, so that consecutive work-groups (XCDs in turn) take one each and an L2 holds few heads' rows.
    const int h = index % a.cache.n_kv_heads, rest = index / a.cache.n_kv_heads;
    const int block = rest % a.blocks, piece = rest / a.blocks;
    const int begin = piece * a.chunk, end = min(begin + a.chunk, a.prefix_len);
    const int rows = prefix_rows(a), H_q = a.cache.n_kv_heads * a.group;

    u32x4* const lk = reinterpret_cast<u32x4*>(lds) + (size_t)team * 2 * KEYS * NCH;
    u32x4* const lv = lk + KEYS * NCH;
    using Tile = Staged<D, E4M3, TEAM, false>;
    if (begin + team * KEYS < end) Tile::load(first, a, a.prefix_b, h, begin + team * KEYS, end, t);

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
        if (key0 < end) odd |= Tile::store(first, lk, lv, t);
        if (key0 + kRoundKeys < end) Tile::load(first, a, a.prefix_b, h, key0 + kRoundKeys, end, t);
        if (round + kRoundKeys >= end) last();
        if constexpr (TEAM > 1) lds_barrier();
        else lds_done();
        for (int k = 0; k < KEYS && key0 + k < hi; k += 32) attend<D>(r, lk + k * NCH, lv + k * NCH, key0 + k, a.scale_log2);
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
    f32x4* const lds_o = reinterpret_cast<f32x4*>(lds);
    const float l = pair_sum32(r.l);
    lds_barrier();  // (the tiles are read)
#pragma unroll
    for (int m = 0; m < D / 32; ++m)
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
            lds_o[(wave * 32 + col) * WORDS + ((8 * m + 2 * i4 + (lane >> 5)) ^ (col & (WORDS - 1)))] =
                f32x4{r.o[m][4 * i4], r.o[m][4 * i4 + 1], r.o[m][4 * i4 + 2], r.o[m][4 * i4 + 3]};
    if (lane < 32) lds_ml[wave * 32 + lane] = make_float2(r.m, l);
    lds_barrier();
    const int row0 = block * TEAM * 32;
    const size_t to = ((size_t)piece * a.cache.n_kv_heads + h) * rows + row0;
    constexpr int THREADS = kWaves * 64, EACH = TEAM * 32 * WORDS / THREADS;
    const int word = threadIdx.x % WORDS;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int at = (i * THREADS + threadIdx.x) / WORDS;  // row of the block
        float2 ml[TEAMS];
        f32x4 v[TEAMS];
#pragma unroll
        for (int k = 0; k < TEAMS; ++k) {
            ml[k] = lds_ml[k * TEAM * 32 + at];
            v[k] = lds_o[(k * TEAM * 32 + at) * WORDS + (word ^ (at & 31 & (WORDS - 1)))];
        }
        float M = ml[0].x;
#pragma unroll
        for (int k = 1; k < TEAMS; ++k) M = fmaxf(M, ml[k].x);
        const float base = softmax_base(M);
        f32x4 O = v[0];
        float L = ml[0].y;
        if constexpr (TEAMS > 1) {
            O = f32x4{0.f, 0.f, 0.f, 0.f};
            L = 0.f;
        }
#pragma unroll
        for (int k = 0; k < (TEAMS > 1 ? TEAMS : 0); ++k) {
            const float f = fast_exp2(ml[k].x - base);
            L = fmaf(f, ml[k].y, L);
#pragma unroll
            for (int j = 0; j < 4; ++j) O[j] = fmaf(f, v[k][j], O[j]);
        }
        if (row0 + at < rows) {
            reinterpret_cast<f32x4*>(a.part_o)[(to + at) * WORDS + word] = O;
            if (word == 0) reinterpret_cast<float2*>(a.part_ml)[to + at] = make_float2(M, L);
        }
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
    if (side) lv[key * LANES + v_chunk_own<D>(key, at)] = w;
    else lk[key * LANES + k_chunk<D>(key, at)] = w;
}

// Up to 16 heads of a group over some keys, 32 at a time, as columns:
//   S^T [16 keys x 16] = K . Q^T, O^T [D x 16] += V^T [D x 32 keys] . P^T by v_mfma_f32_16x16x32_bf16,
// which needs half the registers of 32 rows.  Lane (m, g) has head m.
template <int D>
struct Heads {
    static constexpr int NCH = D / 8;
    u32x4 q[D / 32];
    f32x4 o[D / 16];
    float top, sum;

    __device__ __forceinline__ void open(const PrefixArgs& a, int b, int h, int m, int g) {
        const u32x4* const from =
            reinterpret_cast<const u32x4*>(a.q + ((size_t)b * a.cache.n_kv_heads * a.group + h * a.group + (m < a.group ? m : 0)) * D);
#pragma unroll
        for (int s = 0; s < D / 32; ++s) q[s] = from[4 * s + g];
#pragma unroll
        for (int t = 0; t < D / 16; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        top = -INFINITY;
        sum = 0.f;
    }
    // The first `left` of the 32 keys in LDS.
    __device__ __forceinline__ void step(const u32x4* lk, const u32x4* lv, int left, float scale_log2, int m, int g) {
        float s[8];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < D / 32; ++st) acc = mfma16(lk[(16 * kt + m) * NCH + k_chunk<D>(m, 4 * st + g)], q[st], acc);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * kt + i] = 16 * kt + i < left - 4 * g ? acc[i] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
        const float cand = fmaxf(top, pair_max32(pair_max16(mx)) * scale_log2);
        if (__ballot(cand > top + kRescaleSlack) != 0) {
            const float corr = cand == -INFINITY ? 1.f : fast_exp2(top - cand);
            top = cand;
            sum *= corr;
#pragma unroll
            for (int t = 0; t < D / 16; ++t) o[t] *= corr;
        }
        const float shift = softmax_base(top);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            s[i] = fast_exp2(fmaf(s[i], scale_log2, -shift));
            sum += s[i];
        }
        // The lane's keys of both products: 4 g .. 4 g + 3 of either half.
        const u32x4 p = {pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]), pack_bf16x2(s[4], s[5]), pack_bf16x2(s[6], s[7])};
        const int key = 4 * g + (m >> 2);
        const uint8_t* const base = reinterpret_cast<const uint8_t*>(lv) + key * (2 * D) + 8 * (m & 1);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
            const uint8_t* const v = base + 16 * v_chunk_own<D>(key, 2 * t + ((m >> 1) & 1));
            const u32x2 v0 = lds_read_tr16(v), v1 = lds_read_tr16(v + 16 * (2 * D));
            o[t] = mfma16(u32x4{v0[0], v0[1], v1[0], v1[1]}, p, o[t]);
        }
    }
    __device__ __forceinline__ float l() const { return pair_sum32(pair_sum16(sum)); }
};

// The appended row of sequence b: inside the cache, and not among the prefix's rows, which others are reading; or -1.
__device__ __forceinline__ int appended_row(const PrefixArgs& a, int b) {
    if (a.k_new == nullptr || b >= a.batch) return -1;
    const int pos = a.positions[b];
    return pos < 0 || pos >= a.cache.l_max || (b == a.prefix_b && pos < a.prefix_len) ? -1 : pos;
}

// A wave's run of own rows as one stream of steps of 32 keys.  Two steps' loads are under way while one is worked on.
template <int D, bool E4M3>
struct OwnRows {
    static constexpr int NCH = D / 8;
    struct Step {
        int b, h, L, key, pos;
        bool opens, closes, there;  // the first and last of a part; whether there is such a step
    };
    const PrefixArgs& a;
    u32x4 *lk, *lv;
    size_t part0;
    int lane, m, g, n_waves, me;
    int wave, left;  // the wave's place among the runs; steps left behind the last one issued
    // A window of 64 sequences, one a lane: own rows and the appended row.
    int c0 = -64, len = 0, pos_of = -1;
    Step at[2], ahead;  // what the two loads under way are for; the last one issued
    Loaded<D, E4M3> staged[2];
    Heads<D> rows;  // the part's

    __device__ __forceinline__ OwnRows(const PrefixArgs& args, int index, int prefix_wgs, int wgs, uint8_t* lds) : a(args) {
        lane = threadIdx.x & 63;
        m = lane & 15;
        g = lane >> 4;
        const int in_wg = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        lk = reinterpret_cast<u32x4*>(lds) + (size_t)in_wg * 2 * kOwnKeys * NCH;
        lv = lk + kOwnKeys * NCH;
        part0 = (size_t)a.pieces * a.cache.n_kv_heads * prefix_rows(a);
        n_waves = wgs * kWaves;
        me = in_wg * wgs + index;
        const Runs runs(a, prefix_wgs, wgs, 0);
        wave = index >= prefix_wgs ? in_wg * (wgs - prefix_wgs) + index - prefix_wgs : runs.others + in_wg * prefix_wgs + index;
        const int begin = runs.begin(wave);
        left = wave < runs.others ? runs.first : runs.rest;
        ahead.there = left > 0 && find(begin);
        finish();
        at[0] = ahead;
        forward();
        at[1] = ahead;
    }
    __device__ __forceinline__ void window(int from) {
        c0 = from;
        len = own_len(a, c0 + lane);
        pos_of = appended_row(a, c0 + lane);
    }
    __device__ __forceinline__ void take(int i) {  // the window's i-th sequence
        ahead.b = c0 + i;
        ahead.L = __builtin_amdgcn_readlane(len, i);
        ahead.pos = __builtin_amdgcn_readlane(pos_of, i);
    }
    // Sets `ahead` to the step that lies `to` steps behind the first of all; false: there are not so many.
    __device__ __forceinline__ bool find(int to) {
        int before = 0;
        for (int from = 0; from < a.batch; from += 64) {
            window(from);
            const int upto = before + wave_scan(own_steps(len)) * a.cache.n_kv_heads;
            const unsigned long long past = __ballot(upto > to);
            if (past != 0) {
                const int i = (int)__builtin_ctzll(past);
                take(i);
                const int each = own_steps(ahead.L);
                const int in = to - (__builtin_amdgcn_readlane(upto, i) - each * a.cache.n_kv_heads);
                ahead.h = in / each;
                ahead.key = (in - ahead.h * each) * kOwnKeys;
                ahead.opens = true;
                return true;
            }
            before = __builtin_amdgcn_readlane(upto, 63);
        }
        return false;
    }
    __device__ __forceinline__ void finish() {
        left -= 1;
        ahead.closes = left == 0 || ahead.key + kOwnKeys >= ahead.L;
    }
    __device__ __forceinline__ void forward() {
        if (!ahead.there) return;
        ahead.there = left > 0;
        if (!ahead.there) return;
        ahead.key += kOwnKeys;
        ahead.opens = ahead.key >= ahead.L;
        if (ahead.opens) {
            ahead.key = 0;
            if (++ahead.h == a.cache.n_kv_heads) {
                ahead.h = 0;
                unsigned long long next = __ballot(len > 0 && lane > ahead.b - c0);
                while (next == 0) {
                    if (c0 + 64 >= a.batch) {
                        ahead.there = false;
                        return;
                    }
                    window(c0 + 64);
                    next = __ballot(len > 0);
                }
                take((int)__builtin_ctzll(next));
            }
        }
        finish();
    }
    __device__ __forceinline__ void append() const {
        if (a.k_new == nullptr) return;
        for (int u = me; u < a.batch * a.cache.n_kv_heads; u += n_waves) {
            const int b = u / a.cache.n_kv_heads, pos = appended_row(a, b);
            if (pos >= 0) append_row<D, E4M3>(a, b, u - b * a.cache.n_kv_heads, pos);
        }
    }
    template <int I>
    __device__ __forceinline__ void load() {
        if (at[I].there) Staged<D, E4M3, 1, true>::load(staged[I], a, at[I].b, at[I].h, at[I].key, at[I].L, lane);
    }
    template <int I>
    __device__ __forceinline__ void step() {
        const Step now = at[I];
        if (now.opens) rows.open(a, now.b, now.h, m, g);
        asm volatile("" ::: "memory");  // (the tile before is read)
        Staged<D, E4M3, 1, true>::store(staged[I], lk, lv, lane);
        forward();
        at[I] = ahead;
        load<I>();
        if (now.pos >= now.key && now.pos < now.key + kOwnKeys && now.pos < now.L) {
            lds_done();
            put_row<D, E4M3>(a, now.b, now.h, now.pos - now.key, lk, lv);
        }
        lds_done();
        rows.step(lk, lv, now.L - now.key, a.scale_log2, m, g);
        if (now.closes) {
            const float l = rows.l();
            const size_t row = part0 + ((size_t)now.b * a.cache.n_kv_heads + now.h + wave) * a.group + m;
            if (m < a.group) {
#pragma unroll
                for (int t = 0; t < D / 16; ++t) reinterpret_cast<f32x4*>(a.part_o + row * D)[4 * t + g] = rows.o[t];
                if (g == 0) reinterpret_cast<float2*>(a.part_ml)[row] = make_float2(rows.top, l);
            }
        }
    }
    __device__ __forceinline__ void run() {
        while (at[0].there) {
            step<0>();
            if (!at[1].there) break;
            step<1>();
        }
    }
};

// ---- the launches --------------------------------------------------------------------------------------------

template <int D, bool E4M3, int TEAM>
__global__ __launch_bounds__(kWaves * 64, 2) void decode_prefix_kernel(PrefixArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[tile_bytes<D>()];
    __shared__ float2 lds_ml[kWaves * 32];
    __shared__ int lds_odd[kWaves];
    // A work-group has a part of the prefix, if there are so many, and then some of the own rows.
    const int prefix_wgs = a.pieces * a.blocks * a.cache.n_kv_heads, wgs = max(prefix_wgs, a.own_wgs), index = wide_block();
    if (index >= wgs) return;
    OwnRows<D, E4M3> own(a, index, prefix_wgs, wgs, lds);
    if (index < prefix_wgs) {
        prefix_task<D, E4M3, TEAM>(a, index, lds, lds_ml, lds_odd, own.staged[0], [&]() __attribute__((always_inline)) { own.template load<0>(); });
    } else {
        own.template load<0>();
    }
    own.template load<1>();
    own.append();
    own.run();
}

// Short prefixes and contexts, few sequences: a work-group per (sequence, kv head) takes all of its keys, the prefix's first,
// wave by wave in steps of 32, and its waves meet in LDS.  No partials and one launch; the prefix is read once a sequence.
template <int D, bool E4M3>
__global__ __launch_bounds__(kWholeWaves * 64, 2) void decode_prefix_whole_kernel(PrefixArgs a) {
    constexpr int NCH = D / 8, WORDS = D / 4;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kWholeWaves * 2 * kOwnKeys * D * 2];
    __shared__ float2 lds_ml[kWholeWaves * 16];
    const int unit = wide_block(), b = unit / a.cache.n_kv_heads, h = unit - b * a.cache.n_kv_heads;
    if (b >= a.batch) return;
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int L = own_len(a, b), pos = appended_row(a, b);
    const int shared = b == a.prefix_b ? 0 : a.shared != nullptr ? max(min(a.shared[b], a.prefix_len), 0) : a.prefix_len;
    const int n_prefix = own_steps(shared), n = n_prefix + own_steps(L);
    u32x4* const lk = reinterpret_cast<u32x4*>(lds) + (size_t)wave * 2 * kOwnKeys * NCH;
    u32x4* const lv = lk + kOwnKeys * NCH;
    using Tile = Staged<D, E4M3, 1, true>;
    Loaded<D, E4M3> staged[2];
    auto load = [&](Loaded<D, E4M3>& x, int s) __attribute__((always_inline)) {
        if (s >= n) return;
        const bool own = s >= n_prefix;
        Tile::load(x, a, own ? b : a.prefix_b, h, kOwnKeys * (own ? s - n_prefix : s), own ? L : shared, lane);
    };
    load(staged[0], wave);
    load(staged[1], wave + kWholeWaves);
    Heads<D> rows;
    rows.open(a, b, h, m, g);
    auto step = [&](Loaded<D, E4M3>& x, int s) __attribute__((always_inline)) {
        const int key = kOwnKeys * (s >= n_prefix ? s - n_prefix : s), left = (s >= n_prefix ? L : shared) - key;
        asm volatile("" ::: "memory");  // (the tile before is read)
        Tile::store(x, lk, lv, lane);
        load(x, s + 2 * kWholeWaves);
        if (s >= n_prefix && pos >= key && pos < key + kOwnKeys && pos < L) {
            lds_done();
            put_row<D, E4M3>(a, b, h, pos - key, lk, lv);
        }
        lds_done();
        rows.step(lk, lv, left, a.scale_log2, m, g);
    };
    for (int s = wave; s < n; s += 2 * kWholeWaves) {
        step(staged[0], s);
        if (s + kWholeWaves >= n) break;
        step(staged[1], s + kWholeWaves);
    }
    if (wave == 0 && pos >= 0) append_row<D, E4M3>(a, b, h, pos);
    // The waves meet: [wave][head] rows of O.
    const float l = rows.l();
    lds_barrier();  // (the tiles are read)
    f32x4* const lds_o = reinterpret_cast<f32x4*>(lds);
    if (m < a.group) {
#pragma unroll
        for (int t = 0; t < D / 16; ++t) lds_o[(wave * 16 + m) * WORDS + ((4 * t + g) ^ m)] = rows.o[t];
        if (g == 0) lds_ml[wave * 16 + m] = make_float2(rows.top, l);
    }
    lds_barrier();
    for (int i = threadIdx.x; i < a.group * WORDS; i += kWholeWaves * 64) {
        const int head = i / WORDS, word = i % WORDS;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWholeWaves; ++w) top = fmaxf(top, lds_ml[w * 16 + head].x);
        const float base = softmax_base(top);
        f32x4 O = {0.f, 0.f, 0.f, 0.f};
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWholeWaves; ++w) {
            const float2 ml = lds_ml[w * 16 + head];
            const f32x4 o = lds_o[(w * 16 + head) * WORDS + (word ^ head)];
            const float f = fast_exp2(ml.x - base);
            sum = fmaf(f, ml.y, sum);
#pragma unroll
            for (int k = 0; k < 4; ++k) O[k] = fmaf(f, o[k], O[k]);
        }
        const size_t row = ((size_t)b * a.cache.n_kv_heads + h) * a.group + head;
        u32x2 w;
        w[0] = pack_bf16x2(softmax_out(O[0], sum), softmax_out(O[1], sum));
        w[1] = pack_bf16x2(softmax_out(O[2], sum), softmax_out(O[3], sum));
        __builtin_memcpy(a.out + row * D + 4 * word, &w, 8);  // (2-byte aligned)
        if (word == 0 && a.lse != nullptr) a.lse[row] = softmax_lse(top, sum);
    }
}

// Joins a query row's partials with log-sum-exp weights: WAVES waves per row, which take them in turn.  A wave has the weights
// of 64 partials in its lanes, and D / 4 lanes for each of the partials that it adds at a time.
constexpr int kMergeWaves = 4;
template <int D, int WAVES>
__global__ __launch_bounds__(kMergeWaves * 64) void decode_prefix_merge_kernel(PrefixArgs a) {
    constexpr int E = D / 4, AT_ONCE = 64 / E, DEEP = 4;
    const int in_wg = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, e = lane % E, of = lane / E;
    const int H_q = a.cache.n_kv_heads * a.group, out_row = wide_block() * (kMergeWaves / WAVES) + in_wg / WAVES, b = out_row / H_q;
    if (b >= a.batch) return;  // (with WAVES > 1 for the whole work-group)
    const int head = out_row - b * H_q, h = head / a.group, g = head - h * a.group;
    const int limit = b == a.prefix_b ? 0 : a.shared != nullptr ? min(a.shared[b], a.prefix_len) : a.prefix_len;
    const int n_prefix = limit > 0 ? (limit + a.chunk - 1) / a.chunk : 0;
    const int prefix_wgs = a.pieces * a.blocks * a.cache.n_kv_heads;
    const Runs runs(a, prefix_wgs, max(prefix_wgs, a.own_wgs), b);
    const int steps = own_steps(own_len(a, b));
    const int first = runs.before * a.cache.n_kv_heads + h * steps;
    const int first_wave = steps > 0 ? runs.wave_of(first) : 0;
    const int n_own = steps > 0 ? runs.wave_of(first + steps - 1) - first_wave + 1 : 0, n = n_prefix + n_own;
    const size_t rows = prefix_rows(a);
    const size_t prefix_row = h * rows + (size_t)(b - (b > a.prefix_b ? 1 : 0)) * a.group + g, prefix_step = a.cache.n_kv_heads * rows;
    const size_t own_row = (size_t)a.pieces * prefix_step + ((size_t)b * a.cache.n_kv_heads + h + first_wave) * a.group + g;
    const size_t own_step = a.group;
    auto row_of = [&](int s) __attribute__((always_inline)) {
        return s < n_prefix ? prefix_row + s * prefix_step : own_row + (s - n_prefix) * own_step;
    };
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    const int mine = n > in_wg % WAVES ? (n - in_wg % WAVES + WAVES - 1) / WAVES : 0;  // partials of this wave
    for (int c0 = 0; c0 < mine; c0 += 64) {
        const int here = min(mine - c0, 64);
        float2 ml = make_float2(-INFINITY, 0.f);
        if (lane < here) ml = reinterpret_cast<const float2*>(a.part_ml)[row_of((c0 + lane) * WAVES + in_wg % WAVES)];
        float top = ml.x;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
        top = fmaxf(M, top);
        const float base = softmax_base(top), keep = fast_exp2(M - base), f = fast_exp2(ml.x - base);
        float l = f * ml.y;
#pragma unroll
        for (int x = 1; x < 64; x *= 2) l += __shfl_xor(l, x);
        L = fmaf(L, keep, l);
        O *= keep;
        M = top;
        for (int i0 = 0; i0 < here; i0 += AT_ONCE * DEEP) {
            f32x4 o[DEEP];
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const int i = i0 + d * AT_ONCE + of;
                o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (i < here) o[d] = reinterpret_cast<const f32x4*>(a.part_o + row_of((c0 + i) * WAVES + in_wg % WAVES) * D)[e];
            }
#pragma unroll
            for (int d = 0; d < DEEP; ++d) {
                const float weight = __shfl(f, (i0 + d * AT_ONCE + of) & 63);
#pragma unroll
                for (int x = 0; x < 4; ++x) O[x] = fmaf(weight, o[d][x], O[x]);
            }
        }
    }
#pragma unroll
    for (int x = E; x < 64; x *= 2)
#pragma unroll
        for (int k = 0; k < 4; ++k) O[k] += __shfl_xor(O[k], x);
    if constexpr (WAVES > 1) {
        __shared__ __attribute__((aligned(16))) f32x4 lds_o[WAVES][E];
        __shared__ float2 lds_ml[WAVES];
        if (of == 0) lds_o[in_wg][e] = O;
        if (lane == 0) lds_ml[in_wg] = make_float2(M, L);
        __syncthreads();
        if (in_wg != 0) return;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, lds_ml[w].x);
        const float base = softmax_base(top);
        O = f32x4{0.f, 0.f, 0.f, 0.f};
        L = 0.f;
        M = top;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = fast_exp2(lds_ml[w].x - base);
            L = fmaf(f, lds_ml[w].y, L);
#pragma unroll
            for (int k = 0; k < 4; ++k) O[k] = fmaf(f, lds_o[w][e][k], O[k]);
        }
    }
    if (of == 0) {
        u32x2 w;
        w[0] = pack_bf16x2(softmax_out(O[0], L), softmax_out(O[1], L));
        w[1] = pack_bf16x2(softmax_out(O[2], L), softmax_out(O[3], L));
        __builtin_memcpy(a.out + (size_t)out_row * D + 4 * e, &w, 8);  // (2-byte aligned)
    }
    if (lane == 0 && a.lse != nullptr) a.lse[out_row] = softmax_lse(M, L);
}

template <int D, bool E4M3>
hipError_t launch_prefix_t(const PrefixArgs& a, const Launch& l) {
    const dim3 grid = wide_grid(std::max<int64_t>((int64_t)a.pieces * a.blocks * a.cache.n_kv_heads, a.own_wgs)), block(kWaves * 64);
    if (a.row_tiles == 4) return launch_kernel(decode_prefix_kernel<D, E4M3, 4>, grid, block, l, a);
    if (a.row_tiles == 2) return launch_kernel(decode_prefix_kernel<D, E4M3, 2>, grid, block, l, a);
    return launch_kernel(decode_prefix_kernel<D, E4M3, 1>, grid, block, l, a);
}

template <int D, bool E4M3>
hipError_t launch_whole_t(const PrefixArgs& a, const Launch& l) {
    return launch_kernel(decode_prefix_whole_kernel<D, E4M3>, wide_grid((int64_t)a.batch * a.cache.n_kv_heads), dim3(kWholeWaves * 64), l, a);
}

}  // namespace

// Whether a work-group per (sequence, kv head) takes all of its keys, which the context's capacity bounds (the lengths are on
// the device): where they are few and every work-group has a CU.  us beside other launches, against pieces and a join, 32
// query heads over 8 of 128: a sequence of 100 rows behind 100 3.5 against 6.2, eight of 300 behind 300 4.1 / 6.4, eight of 500 behind
// 500 5.8 / 6.9 (alone 25.5 / 24.7 with the host's share), but four of 1000 behind 1000 9.4 / 7.2; 8 over 2 heads of 64,
// 1000 behind 1000 5.0 / 6.4.
bool prefix_whole(int head_dim, const PrefixArgs& a, int n_cu) {
    return (int64_t)a.batch * a.cache.n_kv_heads <= n_cu && ((int64_t)a.prefix_len + a.cache.l_max) * head_dim <= kWholeValues;
}

hipError_t launch_decode_prefix_whole(int head_dim, const PrefixArgs& a, const Launch& l) {
    const bool e4m3 = a.cache.k_scale != nullptr;
    if (head_dim == 128) return e4m3 ? launch_whole_t<128, true>(a, l) : launch_whole_t<128, false>(a, l);
    if (head_dim == 64) return e4m3 ? launch_whole_t<64, true>(a, l) : launch_whole_t<64, false>(a, l);
    return hipErrorInvalidValue;
}

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
    a->own_wgs = 2 * n_cu;
}

int64_t prefix_partial_rows_max(int batch, int n_kv_heads, int group, int n_cu) {
    PrefixArgs a{};
    a.batch = batch;
    a.group = group;
    a.cache.n_kv_heads = n_kv_heads;
    plan_prefix(&a, n_cu);
    const int64_t pieces = most_pieces(a, n_cu), wgs = std::max<int64_t>(pieces * a.blocks * n_kv_heads, a.own_wgs);
    return pieces * n_kv_heads * batch * group + ((int64_t)batch * n_kv_heads + wgs * kWaves) * group;
}

hipError_t launch_decode_prefix(int head_dim, const PrefixArgs& a, const Launch& l) {
    const bool e4m3 = a.cache.k_scale != nullptr;
    if ((int64_t)a.pieces * a.blocks * a.cache.n_kv_heads > INT32_MAX / kWaves) return hipErrorInvalidValue;
    if (head_dim == 128) return e4m3 ? launch_prefix_t<128, true>(a, l) : launch_prefix_t<128, false>(a, l);
    if (head_dim == 64) return e4m3 ? launch_prefix_t<64, true>(a, l) : launch_prefix_t<64, false>(a, l);
    return hipErrorInvalidValue;
}

hipError_t launch_decode_prefix_merge(int head_dim, const PrefixArgs& a, int n_cu, const Launch& l) {
    const int64_t rows = (int64_t)a.batch * a.cache.n_kv_heads * a.group;
    if (rows > INT32_MAX - kMergeWaves) return hipErrorInvalidValue;
    // A wave per row where that makes a work-group for each CU: 7.8 us for 64 sequences of 32 heads and some 20 partials (with
    // four waves per row 12.0); four waves where rows are few and may have hundreds: 8.4 us for 16 such sequences behind
    // 65536 rows and with 4096 to 8192 of their own (a wave per row 14.0), 13 us for two with 32768 (41).
    const bool many = rows >= (int64_t)kMergeWaves * n_cu;
    const dim3 grid = wide_grid(many ? (rows + kMergeWaves - 1) / kMergeWaves : rows), block(kMergeWaves * 64);
    if (head_dim == 128) {
        if (many) return launch_kernel(decode_prefix_merge_kernel<128, 1>, grid, block, l, a);
        return launch_kernel(decode_prefix_merge_kernel<128, kMergeWaves>, grid, block, l, a);
    }
    if (head_dim == 64) {
        if (many) return launch_kernel(decode_prefix_merge_kernel<64, 1>, grid, block, l, a);
        return launch_kernel(decode_prefix_merge_kernel<64, kMergeWaves>, grid, block, l, a);
    }
    return hipErrorInvalidValue;
}

}  // namespace lara
