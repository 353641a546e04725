// Split-KV GQA decode over the E4M3 cache (kv8_device.h has the rows' format), gfx950.
//
// With K and V rows of codes c, c' and scales 2^a, 2^b, for one query row:
//   s_k = scale * 2^a_k * sum_d q[d] c_k[d]      p_k = exp(s_k - m)
//   O   = sum_k (p_k 2^b_k) c'_k,  l = sum_k p_k,  out = bf16(O / l)
// An E4M3 value is exact in bf16, so the products run on the bf16 matrix cores with Q unrounded; K's scale comes with the
// conversion (v_cvt_scalef32_pk_bf16_fp8), V's multiplies p (by a power of two: exact) before p is rounded to bf16, the
// one rounding of the operands (half a step, 2^-8 of p at most).  Sums, maxima and O are fp32.
//
// Direct launches (a small grid): the keys of every (sequence, kv head) are cut into pieces of `chunk` keys, a work-group
// each.
// Shares (the others): the pieces of all (sequence, kv head)s, in order, are cut into one run per work-group, of equal
// cost to within a piece whatever the lengths are.  A run is a few segments: the end of one (sequence, kv head), whole
// ones, the beginning of another.  Whole ones are written as they end; the others leave fp32 partials (O, m, l), at most
// two a work-group, that meet with log-sum-exp weights in a second launch -- those of a direct launch in the launch itself
// where it is small (by the last work-group of a (sequence, kv head) to arrive).  Every K/V byte is read once for all
// heads of the group.
//
// What bounds it: memory.  64 x 8192 keys, 8 kv heads of 128 (1.08 GB): 155 us, 6.98 TB/s (a read of 1 GiB: 7.02); 61
// sequences of 512 .. 8192 keys over 64-row pages and three idle slots (549 MB): 90 us beside other launches, 6.1 TB/s, 100
// .. 112 alone; one of 4097 keys in a cache of as many (8.5 MB): 4.7 / 10.4, the latency of the launch, one round of loads and the
// merge.  Pieces of a direct launch follow from the cache's rows, not from the lengths, so a short sequence in a large
// cache has few: the same 4097 keys in 8192 rows 6.6 / 11.1, in 32768 9.8 / 16.2, in 131072 12.1 / 35.4.
//
// Inside a segment the waves take rounds of keys in turn (four waves 64, eight 32: small launches, which are one latency
// chain), the next round's K being loaded once the scores are
// out and its V after the second product -- across segments too, with the next segment's Q.  There is no LDS in the
// loop, where the bf16 kernel passes K and V through it:
//   S^T [16 keys x 16 heads] = K . Q^T, by tiles.  Lane (m, g) = (l % 16, l / 16) loads the 16-byte chunks
//     g, g + 4 of key m's row, which are operand A as they lie: the order of the dims inside the sum is free, so half of
//     a chunk is the 8 values that lane gives one v_mfma_f32_16x16x32_bf16, and Q is loaded in the same order.
//   The result leaves lane (m, g) the scores of keys 4g .. 4g + 3 of each tile for head m: the softmax is per lane, and
//     the 8 p of two tiles are operand B of the second product, slots u = 0 .. 7 for keys 16 (u / 4) + 4g + u % 4.
//   O^T [D x 16 heads] += V^T . P^T.  Eight lanes load a row of V, lane (m, g) D / 8 codes (dims D/8 * (m % 8) ..) of key
//     4g + 2e + m / 8 (whole 128-byte lines: rows loaded by 16 lanes, 8 bytes each, streamed at 6.4 TB/s against 6.85, a
//     plain read of 1 GiB); then lanes m and m + 8 exchange halves, so that m < 8 has the first D / 16 dims of both keys,
//     m >= 8 the others.  Byte t of them belongs to row m of tile t, dim D/16 * (2 (m % 8) + m / 8) + t.  v_perm_b32 pairs
//     the bytes of two keys, the conversion makes them a word of operand A.
// A row of length 0 writes zeros and -inf, one with a score of NaN writes NaN.  Rows past a sequence's end are cleared (a
// stale code may be NaN, and 0 * NaN is NaN) and their scores masked.
//
// The row appended by the launch: the wave whose round holds it quantises it for itself, puts it into the round's
// registers and writes it to the cache, so no wave waits for another.
#include "decode_common.h"
#include "kv8_device.h"

#include <math.h>

#include <type_traits>

namespace lara {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kMergeParts = 4;   // a head's partials are summed as s % 4 apart, then these four in order
constexpr int kPartBatch = 4;  // partials in flight of one part

__device__ __forceinline__ f32x4 mfma_bf16(const u32x4& a, const u32x4& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

// Two codes (the low or high half of `codes`) times 2^k, as a word of bf16.
template <bool HIGH>
__device__ __forceinline__ uint32_t codes_to_bf16(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
}

// The word of the lane 8 further in a row of 16 lanes.
__device__ __forceinline__ uint32_t swap_halves(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, true);  // row_ror:8
}

template <bool CACHED, typename T>
__device__ __forceinline__ T load_stream(const void* p) {
    if constexpr (CACHED) return *reinterpret_cast<const T*>(p);
    else return __builtin_nontemporal_load(reinterpret_cast<const T*>(p));
}

// ---- shares --------------------------------------------------------------------------------------------

// Pieces of L keys (DecodeArgs::chunk is a power of two here): a last one of at most a quarter joins the one before it.
__device__ __forceinline__ int pieces_of(const DecodeArgs& a, int L) {
    const int n = (L + a.chunk - 1) >> a.chunk_log2;
    return n <= 1 ? 1 : L - ((n - 1) << a.chunk_log2) <= a.chunk / 4 ? n - 1 : n;
}

// Runs are cut by cost, in quarter pieces: a (sequence, kv head) of n pieces costs 4 n + kOverhead (a segment's waves meet
// and hand over, which takes about as long as three quarters of a piece under load), piece k of it lies at kOverhead + 4 k,
// and work-group w takes the pieces that lie in w * run .. (w + 1) * run - 1 (run >= 4).
constexpr int kOverhead = 3;

// 64 sequences' lengths and appended rows, one per lane.
struct Window {
    int c0 = -1, len = 0, pos = -1;
    __device__ __forceinline__ void load(const DecodeArgs& a, int b) {  // so that it holds sequence b (wave-uniform)
        if (c0 >= 0 && b >= c0 && b < c0 + 64) return;
        c0 = b & ~63;
        const int s = c0 + (threadIdx.x & 63);
        len = s < a.batch ? clamp_len(a.lens[s], a.l_max) : 0;
        pos = s < a.batch && a.k_new != nullptr ? a.positions[s] : -1;
    }
    // Cost of this lane's sequence, all kv heads (0 past the batch).
    __device__ __forceinline__ int cost(const DecodeArgs& a) const {
        return c0 + (int)(threadIdx.x & 63) < a.batch ? a.n_kv_heads * (4 * pieces_of(a, len) + kOverhead) : 0;
    }
};

template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_dpp(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
// Inclusive prefix sums over the wave's lanes (all active).
__device__ __forceinline__ int wave_scan(int v) {
    v = scan_dpp<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8
    v = scan_dpp<0x112, 0xF>(v);
    v = scan_dpp<0x114, 0xF>(v);
    v = scan_dpp<0x118, 0xF>(v);
    v = scan_dpp<0x142, 0xA>(v);  // row_bcast:15, rows 1 and 3
    return scan_dpp<0x143, 0xC>(v);  // row_bcast:31, rows 2 and 3
}

// Cost of a run: the batch's over `runs` work-groups.  Leaves a window of the batch's last part.
__device__ __forceinline__ int run_cost(const DecodeArgs& a, int runs, Window& w) {
    int total = 0;
    for (int c0 = 0; c0 < a.batch; c0 += 64) {
        w.load(a, c0);
        total += __builtin_amdgcn_readlane(wave_scan(w.cost(a)), 63);
    }
    const int run = (total + runs - 1) / runs;
    return run < 4 ? 4 : run;
}

// The sequence in whose cost `at` lies, and the cost before it; -1 past the end.
__device__ __forceinline__ int find_sequence(const DecodeArgs& a, int at, int* before, Window& w) {
    int sum = 0;
    for (int c0 = 0; c0 < a.batch; c0 += 64) {
        w.load(a, c0);
        const int mine = w.cost(a), upto = sum + wave_scan(mine);
        const unsigned long long past = __ballot(mine > 0 && upto > at);
        if (past != 0) {
            const int l = __builtin_ctzll(past);
            *before = __builtin_amdgcn_readlane(upto - mine, l);
            return c0 + l;
        }
        sum = __builtin_amdgcn_readlane(upto, 63);
    }
    return -1;
}

// The partials of a (sequence, kv head), rows of part_o and part_ml for its first head: the first one's, and that of the
// s-th of the others.
struct Partials {
    int n;
    size_t row0, rest, step;
    // Direct launches: one per piece.
    __device__ static Partials direct(const DecodeArgs& a, int unit, int pieces) {
        const size_t row = (size_t)unit * a.max_splits * a.group;
        return Partials{pieces, row, row, (size_t)a.group};
    }
    // Runs: one per work-group that has some of its `pieces`, which lie behind a cost of `base`; in the work-group's slot 0
    // if its run begins with one of them, else in slot 1.
    __device__ static Partials shared(const DecodeArgs& a, int base, int pieces, int run) {
        const int first = (base + kOverhead) / run, last = (base + kOverhead + 4 * (pieces - 1)) / run;
        const int slot = base - 4 < first * run ? 0 : 1;  // (the piece before it lies at base - 4)
        const size_t rest = (size_t)first * 2 * a.group;
        return Partials{last - first + 1, rest + (size_t)slot * a.group, rest, (size_t)2 * a.group};
    }
    __device__ size_t row(int s, int g) const { return (s == 0 ? row0 : rest + s * step) + g; }
};

// ---- partials ------------------------------------------------------------------------------------------

// Sums part `part` (partials part, part + 4, ...) of head g: D / 4 lanes, four dims each, at most kPartBatch partials
// per memory round trip.  (M, L) and O against the part's own maximum.
template <int D>
__device__ __forceinline__ void merge_part(const DecodeArgs& a, const Partials& from, int g, int part, float2* ml_out, f32x4* o_out) {
    const int e = threadIdx.x % (D / 4);
    float M = -INFINITY, L = 0.f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = part; s0 < from.n; s0 += kMergeParts * kPartBatch) {
        f32x4 o[kPartBatch];
        float2 w[kPartBatch];
#pragma unroll
        for (int j = 0; j < kPartBatch; ++j) {
            const int s = s0 + j * kMergeParts;
            w[j] = make_float2(-INFINITY, 0.f);
            o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (s < from.n) {
                const size_t row = from.row(s, g);
                w[j] = reinterpret_cast<const float2*>(a.part_ml)[row];
                o[j] = reinterpret_cast<const f32x4*>(a.part_o + row * D)[e];
            }
        }
        float m = M;
#pragma unroll
        for (int j = 0; j < kPartBatch; ++j) m = fmaxf(m, w[j].x);
        const float base = softmax_base(m);
        const float corr = fast_exp2(M - base);  // 0 while M = -inf
        L *= corr;
        O *= corr;
#pragma unroll
        for (int j = 0; j < kPartBatch; ++j) {
            const float f = fast_exp2(w[j].x - base);  // 0 past the last
            L = fmaf(f, w[j].y, L);
#pragma unroll
            for (int i = 0; i < 4; ++i) O[i] = fmaf(f, o[j][i], O[i]);
        }
        M = m;
    }
    *ml_out = make_float2(M, L);
    *o_out = O;
}

// The parts of `heads` heads (g0 ..) of one (sequence, kv head), D / 4 threads each, into LDS, then the output rows.
template <int D>
__device__ __forceinline__ void merge_heads(const DecodeArgs& a, const Partials& from, int b, int h, int g0, int heads,
                                            float* lds_o, float2* lds_ml, int threads) {
    constexpr int E = D / 4;
    for (int task = threadIdx.x / E; task < heads * kMergeParts; task += threads / E) {
        float2 ml;
        f32x4 o;
        merge_part<D>(a, from, g0 + task / kMergeParts, task % kMergeParts, &ml, &o);
        reinterpret_cast<f32x4*>(lds_o)[task * E + threadIdx.x % E] = o;
        if (threadIdx.x % E == 0) lds_ml[task] = ml;
    }
    __syncthreads();
    const int H_q = a.n_kv_heads * a.group;
    for (int idx = threadIdx.x; idx < heads * D; idx += threads) {
        const int g = idx / D, d = idx - g * D;
        const float2* const ml = lds_ml + g * kMergeParts;
        const float M = fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x));
        const float base = softmax_base(M);
        float O = 0.f, L = 0.f;
#pragma unroll
        for (int p = 0; p < kMergeParts; ++p) {
            const float f = fast_exp2(ml[p].x - base);  // 0 for an empty part
            O = fmaf(f, lds_o[(g * kMergeParts + p) * D + d], O);
            L = fmaf(f, ml[p].y, L);
        }
        const size_t row = (size_t)b * H_q + h * a.group + g0 + g;
        a.out[row * D + d] = f32_to_bf16_rne(softmax_out(O, L));
        if (d == 0 && a.lse != nullptr) a.lse[row] = softmax_lse(M, L);
    }
}

// ---- the kernel ------------------------------------------------------------------------------------------

// A segment of a work-group's run, and the rounds of one wave in it: r = wave + NW * i.  The two that need care -- the one
// with the appended row (index `fresh`), and the last one of a sequence that ends inside it (index `part`) -- come last.
struct Segment {
    int b, h, L, pieces;      // pieces of the (sequence, kv head)
    int base;                 // cost before it
    int r0, r1;               // its pieces that the segment takes
    int k_begin, k_end, pos;  // pos: row appended to the sequence (-1: none)
    int n_mine, n_plain, fresh, part;
};

// Waves of a work-group: eight, of 32-key rounds, in direct launches (one latency chain), else four of 64-key rounds, two
// work-groups a CU.
constexpr int kv8_waves(bool direct) { return direct ? 8 : 4; }

template <int D, bool DIRECT, bool PAGED, bool CACHED>
__global__ __launch_bounds__(kv8_waves(DIRECT) * 64, DIRECT ? 4 : 2) void decode_kv8_kernel(DecodeArgs a) {
    constexpr int NW = kv8_waves(DIRECT), RK = kKv8Piece / NW;
    constexpr int CH = D / 64;   // 16-byte chunks of a K row per lane; words of V codes per lane and key in the product
    constexpr int VB = D / 16;   // V codes per lane and key, O tiles
    constexpr int LANES = D / 8;  // lanes that quantise a row
    constexpr int T = RK / 16;   // score tiles of a round
    static_assert(RK % 32 == 0 && RK <= kKv8RoundKeys, "rounds of whole products");
    typedef uint32_t vword __attribute__((ext_vector_type(D / 32)));  // V codes of a lane's load: D / 8 dims of a key

    const int G = a.group, H_q = a.n_kv_heads * G;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t m16 = lane & 15, grp = lane >> 4;
    const bool lower = (lane & 8) == 0;  // of a row's 16 lanes
    const uint8_t* const kc = reinterpret_cast<const uint8_t*>(a.kc);
    const uint8_t* const vc = reinterpret_cast<const uint8_t*>(a.vc);
    const uint8_t* const zero = reinterpret_cast<const uint8_t*>(a.zero_row);

    Window window;
    int run = 0, run_end = 0;
    // Completes a segment whose b, h, r0, r1, L, pos and pieces are set.
    auto fill = [&](Segment& s) __attribute__((always_inline)) {
        if (s.pos >= a.l_max) s.pos = -1;
        s.k_begin = s.r0 << a.chunk_log2;
        s.k_end = s.r1 == s.pieces ? s.L : s.r1 << a.chunk_log2;
        const int rounds = (s.k_end - s.k_begin + RK - 1) / RK;
        s.n_mine = rounds > wave ? (rounds - wave + NW - 1) / NW : 0;
        const int at = (s.pos - s.k_begin) / RK;
        s.fresh = s.pos >= s.k_begin && s.pos < s.k_end && at % NW == wave ? at / NW : s.n_mine;
        s.part = (s.k_end - s.k_begin) % RK != 0 && s.n_mine > 0 && (rounds - 1) % NW == wave ? s.n_mine - 1 : s.n_mine;
        s.n_plain = s.n_mine - (s.fresh < s.n_mine ? 1 : 0) - (s.part < s.n_mine && s.part != s.fresh ? 1 : 0);
    };
    // The same of a run's segment whose b, h, base and r0 are set; false: it has no piece in the run.
    auto open = [&](Segment& s) __attribute__((always_inline)) -> bool {
        window.load(a, s.b);
        s.L = __builtin_amdgcn_readlane(window.len, s.b & 63);
        s.pos = __builtin_amdgcn_readlane(window.pos, s.b & 63);
        s.pieces = pieces_of(a, s.L);
        const int upto = (run_end - s.base - kOverhead + 3) >> 2;  // pieces that lie before the run's end
        s.r1 = upto < s.pieces ? upto : s.pieces;
        if (s.r1 <= s.r0) return false;
        fill(s);
        return true;
    };
    auto next_segment = [&](Segment& s) __attribute__((always_inline)) -> bool {
        if (DIRECT || s.r1 < s.pieces) return false;  // the run ends inside it
        s.base += 4 * s.pieces + kOverhead;
        s.r0 = 0;
        if (++s.h == a.n_kv_heads) {
            s.h = 0;
            if (++s.b >= a.batch) return false;
        }
        return open(s);
    };
    // First key of the wave's i-th round in the order above.
    auto key_of = [&](const Segment& s, int i) __attribute__((always_inline)) {
        const int index = i < s.n_plain ? i + (i >= s.fresh ? 1 : 0) : i == s.n_plain && s.fresh < s.n_mine ? s.fresh : s.part;
        return s.k_begin + (wave + NW * index) * RK;
    };

    Segment seg;
    if constexpr (DIRECT) {
        seg.b = blockIdx.z;
        seg.h = blockIdx.y;
        seg.base = 0;
        seg.r0 = blockIdx.x;
        seg.r1 = blockIdx.x + 1;
        seg.L = clamp_len(a.lens[seg.b], a.l_max);
        seg.pos = a.k_new != nullptr ? a.positions[seg.b] : -1;
        seg.pieces = pieces_of(a, seg.L);
        if (seg.r0 >= seg.pieces) return;  // (the whole work-group, here and below)
        fill(seg);
    } else {
        run = run_cost(a, gridDim.x, window);
        run_end = ((int)blockIdx.x + 1) * run;
        const int at = blockIdx.x * run;
        int before;
        seg.b = __builtin_amdgcn_readfirstlane(find_sequence(a, at, &before, window));
        if (seg.b < 0) return;  // no pieces left
        const int pieces = pieces_of(a, __builtin_amdgcn_readlane(window.len, seg.b & 63));
        const int cost = 4 * pieces + kOverhead;
        seg.h = (at - before) / cost;
        seg.base = before + seg.h * cost;
        const int inside = at - seg.base - kOverhead;
        seg.r0 = inside <= 0 ? 0 : (inside + 3) >> 2;
        if (seg.r0 == pieces) {  // behind its last piece
            seg.base += cost;
            seg.r0 = 0;
            if (++seg.h == a.n_kv_heads) {
                seg.h = 0;
                if (++seg.b >= a.batch) return;
            }
        }
        if (!open(seg)) return;
    }

    // Paged: 64 consecutive block-table entries of a sequence, one per lane, from page pc_first on.
    int pc_seq = -1, pc_first = 0, pc_val = -1;
    auto page_of = [&](int b, int page_idx) -> int {
        if (b != pc_seq || page_idx - pc_first >= 64 || page_idx < pc_first) {
            pc_seq = b;
            pc_first = page_idx;
            const int i = page_idx + lane;
            pc_val = i < a.max_pages ? a.block_table[(size_t)b * a.max_pages + i] : -1;
        }
        return __builtin_amdgcn_readlane(pc_val, page_idx - pc_first);
    };
    // Rounds start at multiples of 64 and a row's region (a page) has a multiple of 64 rows, so all rows of a round lie
    // inside it.
    struct Source {
        const uint8_t *k, *v, *ks, *vs;  // wave-uniform: the round's first row
    };
    auto round_source = [&](const Segment& s, int key0) __attribute__((always_inline)) -> Source {
        int64_t first;
        if constexpr (PAGED) {
            const int page = page_of(s.b, key0 >> a.page_shift);
            if (page < 0) return Source{zero, zero, zero, zero};  // unmapped: rows of zeros
            first = (((int64_t)page * a.n_kv_heads + s.h) << a.page_shift) + (key0 & ((1 << a.page_shift) - 1));
        } else {
            first = ((int64_t)s.b * a.n_kv_heads + s.h) * a.l_cap + key0;
        }
        return Source{kc + first * D, vc + first * D, a.k_scale + first, a.v_scale + first};
    };
    // One round in a wave's registers: K chunks and scale bytes (one per tile), V codes and scale bytes (four a word).
    u32x4 kr[T][CH];
    vword vr[2 * T];
    uint32_t ks[T], vs[T];
    // Byte offsets of a lane's first K chunk and V word inside a round (32 bits beside a uniform base: local(), so that the
    // compiler keeps them that way instead of as 64-bit addresses).
    const uint32_t k_lane = m16 * D + 16 * grp, v_lane = (4 * grp + (m16 >> 3)) * D + D / 8 * (m16 & 7);
    auto local = [](uint32_t v) __attribute__((always_inline)) {
        asm volatile("" : "+v"(v));
        return v;
    };
    auto load_k = [&](const Source& from) __attribute__((always_inline)) {
        const uint8_t* const k = from.k + local(k_lane);
        const uint8_t* const scale = from.ks + local(m16);
#pragma unroll
        for (int t = 0; t < T; ++t) {
#pragma unroll
            for (int j = 0; j < CH; ++j) kr[t][j] = load_stream<CACHED, u32x4>(k + 16 * t * D + 64 * j);
            ks[t] = scale[16 * t];
        }
    };
    auto load_v = [&](const Source& from) __attribute__((always_inline)) {
        const uint8_t* const v = from.v + local(v_lane);
        const uint8_t* const scale = from.vs + local(4 * grp);
#pragma unroll
        for (int n = 0; n < 2 * T; ++n) vr[n] = load_stream<CACHED, vword>(v + (16 * (n >> 1) + 2 * (n & 1)) * D);
#pragma unroll
        for (int t = 0; t < T; ++t) vs[t] = *reinterpret_cast<const uint32_t*>(scale + 16 * t);
    };
    // A segment's Q^T operand: lane (m, g) holds, for chunk j's half i, dims 16 (g + 4j) + 8i .. of head m (heads past G
    // are cleared as it begins); and the appended row, K's in the first lanes and V's in the next.
    u32x4 qb[2 * CH], new_row = {};
    auto load_q = [&](const Segment& s) __attribute__((always_inline)) {
        const u32x4* qp = reinterpret_cast<const u32x4*>(a.q + ((size_t)s.b * H_q + s.h * G + ((int)m16 < G ? m16 : 0)) * D);
#pragma unroll
        for (int j = 0; j < CH; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) qb[2 * j + i] = qp[2 * (grp + 4 * j) + i];
        if (s.pos >= 0 && lane < 2 * LANES) {
            const uint16_t* const rows = lane < LANES ? a.k_new : a.v_new;
            new_row = reinterpret_cast<const u32x4*>(rows + ((size_t)s.b * a.n_kv_heads + s.h) * D)[lane % LANES];
        }
    };

    // What is loaded next: round `ahead_i` of segment `ahead` (of this wave's rounds; segments without any are passed).
    Segment ahead = seg;
    int ahead_i = -1;
    bool ahead_there = true;
    auto step = [&]() __attribute__((always_inline)) -> Source {
        // (Behind the last round the rows of zeros, which every L2 has: a wait counts the loads behind it, so none of
        // them may be conditional.)
        if (!ahead_there) return Source{zero, zero, zero, zero};
        ++ahead_i;
        while (ahead_i >= ahead.n_mine) {
            if (!next_segment(ahead)) {
                ahead_there = false;
                return Source{zero, zero, zero, zero};
            }
            ahead_i = 0;
        }
        return round_source(ahead, key_of(ahead, ahead_i));
    };
    load_q(seg);
    {
        const Source from = step();
        load_k(from);
        load_v(from);
    }

    __shared__ __attribute__((aligned(16))) uint8_t new_codes[NW][2][D];
    __shared__ uint8_t new_scale[NW][2];
    constexpr int OS = D + 4;  // (bank conflicts)
    extern __shared__ __attribute__((aligned(16))) float lds[];  // [NW][G] rows of OS, then (m, l)
    float* const lds_o = lds;
    float2* const lds_ml = reinterpret_cast<float2*>(lds + NW * G * OS);

    for (bool opening = true;; opening = false) {
#pragma unroll
        for (int i = 0; i < 2 * CH; ++i) qb[i] = (int)m16 < G ? qb[i] : u32x4{0u, 0u, 0u, 0u};
        // The appended row: by the wave whose round holds it, or, where no segment does, by wave 0 of the first one.
        const bool new_here = seg.fresh < seg.n_mine;
        if (new_here || (seg.pos >= seg.L && seg.r0 == 0 && wave == 0)) {
            if (lane < 2 * LANES) {
                const int side = lane / LANES, at = lane % LANES;
                float x[8];
                unpack_bf16x8(new_row, x);
                uint32_t byte;
                const u32x2 c = kv8_quantise<LANES>(x, &byte);
                reinterpret_cast<u32x2*>(new_codes[wave][side])[at] = c;
                if (at == 0) new_scale[wave][side] = (uint8_t)byte;
                const int64_t row = PAGED ? paged_row(a.block_table + (size_t)seg.b * a.max_pages, a.page_shift, a.n_kv_heads, seg.h, seg.pos)
                                          : ((int64_t)seg.b * a.n_kv_heads + seg.h) * a.l_cap + seg.pos;
                if (row >= 0) {  // (unmapped: not written)
                    reinterpret_cast<u32x2*>(const_cast<uint8_t*>(side ? vc : kc) + row * D)[at] = c;
                    if (at == 0) (side ? a.v_scale : a.k_scale)[row] = (uint8_t)byte;
                }
            }
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's own writes, which it alone reads
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        }
        f32x4 o_acc[VB];  // tile t: row 4g + i of head m in register i
#pragma unroll
        for (int t = 0; t < VB; ++t) o_acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        float m_run = -INFINITY, l_lane = 0.f;

        // The wave's i-th round.  CARE: rows past the sequence's end are cleared and masked, the appended row is put in.
        auto round = [&](int i, auto care) __attribute__((always_inline)) {
            constexpr bool CARE = decltype(care)::value;
            const int key0 = CARE ? key_of(seg, i) : 0;
            const Source next = step();
            if constexpr (CARE) {
                const int at = new_here ? seg.pos - key0 : -1;
                const uint32_t m = local(m16), g4 = local(4 * grp);  // (worked out here, not kept for every round)
#pragma unroll
                for (int t = 0; t < T; ++t) {
                    const bool here = at == 16 * t + (int)m;
#pragma unroll
                    for (int j = 0; j < CH; ++j) {
                        const u32x4 w = reinterpret_cast<const u32x4*>(new_codes[wave][0])[g4 / 4 + 4 * j];
                        kr[t][j] = here ? w : kr[t][j];
                    }
                    ks[t] = here ? new_scale[wave][0] : ks[t];
                }
#pragma unroll
                for (int n = 0; n < 2 * T; ++n) {
                    const int key = 16 * (n >> 1) + (int)g4 + 2 * (n & 1) + (int)(m >> 3);
                    const vword w = reinterpret_cast<const vword*>(new_codes[wave][1])[m & 7];
                    vr[n] = key0 + key >= seg.k_end ? vword(0u) : key == at ? w : vr[n];
                }
#pragma unroll
                for (int u = 0; u < 4 * T; ++u) {
                    const uint32_t shift = 8 * (u & 3);
                    const uint32_t other = (vs[u >> 2] & ~(0xFFu << shift)) | ((uint32_t)new_scale[wave][1] << shift);
                    vs[u >> 2] = 16 * (u >> 2) + (int)g4 + (u & 3) == at ? other : vs[u >> 2];
                }
            }
            // S^T, tiles of 16 keys.
            float s[4 * T];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const float scale = kv8_scale(ks[t]);
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < CH; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t lo = kr[t][j][2 * i], hi = kr[t][j][2 * i + 1];
                        const u32x4 ka = {codes_to_bf16<false>(lo, scale), codes_to_bf16<true>(lo, scale),
                                          codes_to_bf16<false>(hi, scale), codes_to_bf16<true>(hi, scale)};
                        acc = mfma_bf16(ka, qb[2 * j + i], acc);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    s[4 * t + i] = !CARE || key0 + 16 * t + 4 * (int)local(grp) + i < seg.k_end ? acc[i] : -INFINITY;
            }
            load_k(next);  // (K's registers are free; V's after the second product)
            float mx = s[0];
#pragma unroll
            for (int u = 1; u < 4 * T; ++u) mx = fmaxf(mx, s[u]);
            mx = pair_max32(pair_max16(mx));
            const float m_cand = fmaxf(m_run, mx * a.scale_log2);
            if (__ballot(m_cand > m_run + kRescaleSlack) != 0) {
                const float corr = m_cand == -INFINITY ? 1.f : fast_exp2(m_run - m_cand);
                m_run = m_cand;
                l_lane *= corr;
#pragma unroll
                for (int t = 0; t < VB; ++t) o_acc[t] *= corr;
            }
#pragma unroll
            for (int u = 0; u < 4 * T; ++u) {
                float p = fast_exp2(fmaf(s[u], a.scale_log2, -m_run));
                if (CARE && s[u] == -INFINITY) p = 0.f;  // (m_run may still be -inf)
                l_lane += p;
                s[u] = p * kv8_scale((vs[u >> 2] >> (8 * (u & 3))) & 0xFFu);
            }
            // O^T += V^T . P^T, 32 keys and two tiles (half a word of codes) at a time.
#pragma unroll
            for (int n = 0; n < T / 2; ++n) {
                const float* const p = s + 8 * n;
                const u32x4 pb = {pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]), pack_bf16x2(p[6], p[7])};
#pragma unroll
                for (int w = 0; w < CH; ++w) {
                    uint32_t even[4], odd[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t mine = vr[4 * n + i][w], far = vr[4 * n + i][CH + w];
                        const uint32_t mine_far = swap_halves(mine), far_far = swap_halves(far);  // (all lanes take part)
                        even[i] = lower ? mine : far_far;
                        odd[i] = lower ? mine_far : far;
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        u32x4 va[2];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t two = __builtin_amdgcn_perm(odd[i], even[i], half ? 0x07030602u : 0x05010400u);
                            va[0][i] = codes_to_bf16<false>(two, 1.f);
                            va[1][i] = codes_to_bf16<true>(two, 1.f);
                        }
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            f32x4& o = o_acc[4 * w + 2 * half + c];
                            o = mfma_bf16(va[c], pb, o);
                        }
                    }
                }
            }
            load_v(next);
        };
        int i = 0;
        for (; i < seg.n_plain; ++i) round(i, std::false_type{});
        for (; i < seg.n_mine; ++i) round(i, std::true_type{});

        // The waves meet; the next segment's Q is on its way meanwhile.
        Segment following = seg;
        const bool more = next_segment(following);
        if (more) load_q(following);
        const float l_head = pair_sum32(pair_sum16(l_lane));
        __syncthreads();  // the last segment's readers are done
        if ((int)m16 < G) {
            float* const to = lds_o + (wave * G + m16) * OS;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < VB; t += 4)
                    *reinterpret_cast<f32x4*>(to + VB * (2 * ((4 * grp + i) & 7) + ((4 * grp + i) >> 3)) + t) =
                        f32x4{o_acc[t][i], o_acc[t + 1][i], o_acc[t + 2][i], o_acc[t + 3][i]};
            if (grp == 0) lds_ml[wave * G + m16] = make_float2(m_run, l_head);
        }
        __syncthreads();
        const bool whole = seg.r1 - seg.r0 == seg.pieces;
        const size_t slot = DIRECT ? (((size_t)seg.b * a.n_kv_heads + seg.h) * a.max_splits + seg.r0) * G
                                   : ((size_t)blockIdx.x * 2 + (opening ? 0 : 1)) * G;  // of a partial
        for (int idx = threadIdx.x; idx < G * D; idx += NW * 64) {
            const int g = idx / D, d = idx - g * D;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, lds_ml[w * G + g].x);
            const float base = softmax_base(M);
            float O = 0.f, Ls = 0.f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float2 ml = lds_ml[w * G + g];
                const float f = fast_exp2(ml.x - base);  // 0 for a wave without rounds
                O = fmaf(f, lds_o[(w * G + g) * OS + d], O);
                Ls = fmaf(f, ml.y, Ls);
            }
            if (whole) {
                const size_t to = (size_t)seg.b * H_q + seg.h * G + g;
                a.out[to * D + d] = f32_to_bf16_rne(softmax_out(O, Ls));
                if (d == 0 && a.lse != nullptr) a.lse[to] = softmax_lse(M, Ls);
            } else {
                const size_t to = slot + g;
                if (DIRECT && a.arrivals != nullptr) {  // agent-scope stores: seen across the XCDs without an L2 write-back
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
        if (DIRECT && !whole && a.arrivals != nullptr) {
            // The last work-group of the (sequence, kv head) to arrive merges its partials: a work-group's are stored
            // before thread 0's release increment, the increment that reads n - 1 acquires the others', and resets the
            // counter.
            const int unit = seg.b * a.n_kv_heads + seg.h;
            const Partials from = Partials::direct(a, unit, seg.pieces);
            __shared__ int is_last;
            __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
            __syncthreads();
            if (threadIdx.x == 0) {
                const int prev = __hip_atomic_fetch_add(&a.arrivals[unit], 1, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT);
                is_last = prev == from.n - 1;
                if (is_last) {
                    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
                    __hip_atomic_store(&a.arrivals[unit], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            }
            __syncthreads();
            if (is_last) {
                static_assert(NW >= kMergeParts, "the merge's LDS is inside the waves'");
                merge_heads<D>(a, from, seg.b, seg.h, 0, G, lds, reinterpret_cast<float2*>(lds + kMergeParts * G * D), NW * 64);
            }
        }
        if (!more) break;
        seg = following;
    }
}

// The merge launch: a work-group per (sequence, kv head, head of the group).
template <int D>
__global__ __launch_bounds__(kMergeParts * D / 4) void decode_kv8_merge_kernel(DecodeArgs a) {
    const int block = wide_block(), unit = block / a.group, g = block - unit * a.group;
    const int b = unit / a.n_kv_heads, h = unit - b * a.n_kv_heads;
    if (b >= a.batch) return;
    Partials from;
    if (a.max_splits > 0) {
        from = Partials::direct(a, unit, pieces_of(a, clamp_len(a.lens[b], a.l_max)));
    } else {
        Window window;
        const int run = run_cost(a, a.runs, window);
        int before = 0;  // cost of the sequences before this one
        for (int c0 = 0; c0 < b; c0 += 64) {
            window.load(a, c0);
            before += __builtin_amdgcn_readlane(wave_scan(c0 + (int)(threadIdx.x & 63) < b ? window.cost(a) : 0), 63);
        }
        window.load(a, b);
        const int pieces = pieces_of(a, __builtin_amdgcn_readlane(window.len, b & 63));
        from = Partials::shared(a, before + h * (4 * pieces + kOverhead), pieces, run);
    }
    if (from.n <= 1) return;  // written by its work-group
    __shared__ __attribute__((aligned(16))) float lds_o[kMergeParts * D];
    __shared__ float2 lds_ml[kMergeParts];
    merge_heads<D>(a, from, b, h, g, 1, lds_o, lds_ml, kMergeParts * D / 4);
}

template <int D, bool DIRECT>
hipError_t launch_kv8_t(const DecodeArgs& a, const Launch& l) {
    constexpr int NW = kv8_waves(DIRECT);
    const dim3 grid = DIRECT ? dim3(a.max_splits, a.n_kv_heads, a.batch) : dim3(a.runs);
    const size_t lds = ((size_t)NW * a.group * (D + 4) + NW * a.group * 2) * sizeof(float);
    void (*const kernel)(DecodeArgs) =
        a.block_table != nullptr ? (a.cached ? decode_kv8_kernel<D, DIRECT, true, true> : decode_kv8_kernel<D, DIRECT, true, false>)
                                 : (a.cached ? decode_kv8_kernel<D, DIRECT, false, true> : decode_kv8_kernel<D, DIRECT, false, false>);
    return launch_kernel_lds(kernel, grid, dim3(NW * 64), lds, l, a);
}

}  // namespace

bool decode_kv8_supported(int head_dim, int group) { return (head_dim == 64 || head_dim == 128) && group >= 1 && group <= 16; }

hipError_t launch_decode_kv8(int head_dim, const DecodeArgs& a, const Launch& l) {
    if (!decode_kv8_supported(head_dim, a.group) || (a.max_splits < 1 && a.runs < 1) || a.chunk < kKv8Piece ||
        a.chunk != 1 << a.chunk_log2)
        return hipErrorInvalidValue;
    if (a.max_splits > 0) return head_dim == 128 ? launch_kv8_t<128, true>(a, l) : launch_kv8_t<64, true>(a, l);
    return head_dim == 128 ? launch_kv8_t<128, false>(a, l) : launch_kv8_t<64, false>(a, l);
}

hipError_t launch_decode_kv8_merge(int head_dim, const DecodeArgs& a, const Launch& l) {
    const dim3 grid = wide_grid((int64_t)a.batch * a.n_kv_heads * a.group), block(kMergeParts * head_dim / 4);
    if (head_dim == 128) return launch_kernel(decode_kv8_merge_kernel<128>, grid, block, l, a);
    if (head_dim == 64) return launch_kernel(decode_kv8_merge_kernel<64>, grid, block, l, a);
    return hipErrorInvalidValue;
}

}  // namespace lara
