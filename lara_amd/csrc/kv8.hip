// The E4M3 K/V cache's rows: quantised as they are written, read back as bf16 (kv8_device.h has the format).
//
// Both are one pass over memory: a write moves 2 D bytes in and D + 1 out per row, a read the reverse; D / 8 lanes hold
// a row, so the row's maximum is three or four lane exchanges and no LDS.
//
// Bound by memory: 8192 tokens of 8 kv heads of 128 read back (50 MB) in 7.5 us beside other launches, 6.7 TB/s (8.7 alone,
// 2.7 of them the launch); 2048 written (12.6 MB) in 3.6 / 4.8, where a launch is most of it.  One 16-byte load a side and
// thread: rows are independent, so the grid is the depth.
#include "kv8_device.h"

namespace lara {
namespace {

constexpr int kKv8Threads = 256;

// Rows of K and V: `source` row i of [B or 1][H_kv][n].  positions == nullptr: rows start .. of sequence b; otherwise row
// positions[s] of sequence s, one each (n = 1; skipped outside 0 .. l_max - 1).
template <int D>
__global__ __launch_bounds__(kKv8Threads) void kv8_write_kernel(Kv8WriteArgs a) {
    constexpr int LANES = D / 8;
    const int64_t i = ((int64_t)wide_block() * kKv8Threads + threadIdx.x) / LANES;
    const int part = threadIdx.x % LANES;
    if (i >= a.n_rows) return;  // (a row's lanes leave together)
    int b = a.b, t;
    const int64_t head = i / a.n;
    int h = (int)head;
    if (a.positions != nullptr) {
        b = h / a.cache.n_kv_heads;
        h -= b * a.cache.n_kv_heads;
        t = a.positions[b];
        if (t < 0 || t >= a.cache.l_max) return;
    } else {
        t = a.start + (int)(i - head * a.n);
    }
    const int64_t row = kv8_row(a.cache, b, h, t);
    if (row < 0) return;
    const u32x4 w[2] = {__builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.k) + i * LANES + part),
                        __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.v) + i * LANES + part)};
    uint8_t* const codes[2] = {a.cache.k, a.cache.v};
    uint8_t* const scales[2] = {a.cache.k_scale, a.cache.v_scale};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        float x[8];
        unpack_bf16x8(w[side], x);
        uint32_t byte;
        const u32x2 c = kv8_quantise<LANES>(x, &byte);
        reinterpret_cast<u32x2*>(codes[side] + row * D)[part] = c;
        if (part == 0) scales[side][row] = (uint8_t)byte;
    }
}

// Rows start .. start + n - 1 of sequence b to [H_kv][out_rows][D] bf16 (rows of an unmapped page: zeros).  E4M3: from
// codes and scales; otherwise from a bf16 cache (the words as they are).  Work-groups take the heads in turn, as those of the
// row-block prefill do that reads the rows next: with 8 heads on the same XCD, out of its L2 (256 rows after 7936: 64.4 -> 62.5 us alone, and 9.5 -> 8.7 for this launch; stores past
// the L2: 73.6).
template <int D, bool E4M3>
__global__ __launch_bounds__(kKv8Threads) void kv_read_kernel(KvReadArgs a) {
    constexpr int LANES = D / 8;
    const uint32_t block = wide_block();
    const int h = block % a.cache.n_kv_heads, part = threadIdx.x % LANES;
    const int64_t at = (int64_t)(block / a.cache.n_kv_heads) * (kKv8Threads / LANES) + threadIdx.x / LANES;
    if (at >= a.n) return;
    const int t = (int)at;
    const int64_t row = kv8_row(a.cache, a.b, h, a.start + t);
    const int64_t to = ((int64_t)h * a.out_rows + t) * LANES + part;
    const uint8_t* const codes[2] = {a.cache.k, a.cache.v};
    const uint8_t* const scales[2] = {a.cache.k_scale, a.cache.v_scale};
    u32x4* const out[2] = {reinterpret_cast<u32x4*>(a.k), reinterpret_cast<u32x4*>(a.v)};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        u32x4 o = {0u, 0u, 0u, 0u};
        if (row >= 0) {
            if constexpr (E4M3) {
                const u32x2 c = reinterpret_cast<const u32x2*>(codes[side] + row * D)[part];
                const float scale = kv8_scale(scales[side][row]);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    // (code * 2^k has 4 significant bits: its upper half is the bf16 word)
                    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], false);
                    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], true);
                    o[2 * w] = (__float_as_uint(lo[0] * scale) >> 16) | (__float_as_uint(lo[1] * scale) & 0xFFFF0000u);
                    o[2 * w + 1] = (__float_as_uint(hi[0] * scale) >> 16) | (__float_as_uint(hi[1] * scale) & 0xFFFF0000u);
                }
            } else {
                o = reinterpret_cast<const u32x4*>(codes[side])[row * LANES + part];
            }
        }
        out[side][to] = o;
    }
}

}  // namespace

hipError_t launch_kv8_write(int head_dim, const Kv8WriteArgs& a, const Launch& l) {
    if (a.n_rows < 1) return hipSuccess;
    const int64_t threads = a.n_rows * (head_dim / 8), wgs = (threads + kKv8Threads - 1) / kKv8Threads;
    if (wgs > 0x7FFFFFFF) return hipErrorInvalidValue;
    const dim3 grid = wide_grid(wgs), block(kKv8Threads);
    if (head_dim == 128) return launch_kernel(kv8_write_kernel<128>, grid, block, l, a);
    if (head_dim == 64) return launch_kernel(kv8_write_kernel<64>, grid, block, l, a);
    return hipErrorInvalidValue;
}

hipError_t launch_kv_read(int head_dim, const KvReadArgs& a, const Launch& l) {
    if (a.n < 1) return hipSuccess;
    const int64_t rows = kKv8Threads / (head_dim / 8), wgs = (a.n + rows - 1) / rows * a.cache.n_kv_heads;
    if (wgs > 0x7FFFFFFF) return hipErrorInvalidValue;
    const dim3 grid = wide_grid(wgs), block(kKv8Threads);
    const bool e4m3 = a.cache.k_scale != nullptr;
    if (head_dim == 128)
        return e4m3 ? launch_kernel(kv_read_kernel<128, true>, grid, block, l, a)
                    : launch_kernel(kv_read_kernel<128, false>, grid, block, l, a);
    if (head_dim == 64)
        return e4m3 ? launch_kernel(kv_read_kernel<64, true>, grid, block, l, a)
                    : launch_kernel(kv_read_kernel<64, false>, grid, block, l, a);
    return hipErrorInvalidValue;
}

}  // namespace lara
