// Products with 4-bit weights: y[t, r] = inv_t * sum_g s[r, g] * sum_{k in g} (c[r, k] - 8) * (x[t, k] * gamma[k]), codes c of
// 0 .. 15, one bf16 scale per row r and group g of 32, 64 or 128 columns, inv_t = 1 / sqrt(mean(x_t^2) + eps) with gamma
// and 1 without.
//
// Packed form (gqa_w4_pack_device; a program packs its weights once): tiles of 16 rows x 128 columns, 1 KiB each, a row
// tile's column blocks in order.  Lane l of a wave owns 16 bytes of a tile: row l % 16, and in dword s its 8 columns
// 32s + 8 (l / 16) .. of the block: nibble j of the dword's low half is column 2j, of its high half 2j + 1.  So a wave
// reads a tile as 1 KiB in a row, dword s is operand A of one v_mfma_f32_16x16x32_bf16 whose 32 columns lie in one group
// (of any size), and (dword >> 4j) & 0x000F000F | 0x43004300 is a pair of bf16 128 + c.  Scales: [row tile][group][16].
// Rows past the matrix have code 8 and scale 0, columns past it scale 0.
//
// The constant 136 = 128 + 8 leaves through a product of its own: one more MFMA with operand A = -136 everywhere, into the
// same accumulator.  Products are exact and summed in fp32, a group at a time, then scaled in fp32.
// x * gamma is rounded to bf16 (operand B; half a step of 2^-8, as the normalised rows of the bf16 stage are).
#include "gqa_internal.h"

#include <math.h>

namespace lara {
namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4Threads = 256;
constexpr int kW4Waves = 8;
constexpr int kW4Tokens = 16;  // of a work-group

__host__ __device__ inline int w4_blocks(int hidden) { return (hidden + 127) / 128; }
__host__ __device__ inline int w4_groups(int hidden, int group) { return w4_blocks(hidden) * (128 / group); }

// codes [rows][hidden / 2] (the even column in the low half of a byte), scales [rows][hidden / group] bf16.
__global__ __launch_bounds__(kW4Threads) void w4_pack_kernel(W4PackArgs a) {
    const int64_t i = (int64_t)blockIdx.x * kW4Threads + threadIdx.x;  // a dword of the packed codes
    const int blocks = w4_blocks(a.hidden), tiles = (a.rows + 15) / 16;
    const int64_t dwords = (int64_t)tiles * blocks * 256;
    if (i < dwords) {
        const int s = (int)(i & 3), lane = (int)(i >> 2) & 63;
        const int64_t tile = i >> 8;
        const int row = (int)(tile / blocks) * 16 + (lane & 15);
        const int col = (int)(tile % blocks) * 128 + 32 * s + 8 * (lane >> 4);
        uint32_t out = 0x88888888u;
        if (row < a.rows && col < a.hidden) {  // (hidden is a multiple of 32)
            const uint8_t* const src = a.codes + ((int64_t)row * a.hidden + col) / 2;
            out = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t two = src[j];
                out |= (two & 15u) << (4 * j) | (two >> 4) << (16 + 4 * j);
            }
        }
        a.packed[i] = out;
    }
    const int groups = w4_groups(a.hidden, a.group), given = a.hidden / a.group;
    if (i < (int64_t)tiles * groups * 16) {
        const int r = (int)(i & 15);
        const int64_t rest = i >> 4;
        const int g = (int)(rest % groups), row = (int)(rest / groups) * 16 + r;
        a.packed_scales[i] = row < a.rows && g < given ? a.scales[(int64_t)row * given + g] : (uint16_t)0;
    }
}

// The packed matrix as bf16 [rows][hidden]: (c - 8) * s, one rounding.
__global__ __launch_bounds__(kW4Threads) void w4_unpack_kernel(W4UnpackArgs a) {
    const int64_t i = (int64_t)blockIdx.x * kW4Threads + threadIdx.x;
    const int blocks = w4_blocks(a.hidden), tiles = (a.rows + 15) / 16;
    if (i >= (int64_t)tiles * blocks * 256) return;
    const int s = (int)(i & 3), lane = (int)(i >> 2) & 63;
    const int64_t tile = i >> 8;
    const int row_tile = (int)(tile / blocks), row = row_tile * 16 + (lane & 15);
    const int col = (int)(tile % blocks) * 128 + 32 * s + 8 * (lane >> 4);
    if (row >= a.rows || col >= a.hidden) return;
    const uint32_t c = a.packed[i];
    const float scale = __uint_as_float(
        (uint32_t)a.packed_scales[((int64_t)row_tile * w4_groups(a.hidden, a.group) + col / a.group) * 16 + (lane & 15)] << 16);
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float even = (float)((int)((c >> (4 * j)) & 15u) - 8) * scale, odd = (float)((int)((c >> (16 + 4 * j)) & 15u) - 8) * scale;
        const bf16x2_t pair = {(__bf16)even, (__bf16)odd};
        o[j] = __builtin_bit_cast(uint32_t, pair);
    }
    *reinterpret_cast<u32x4*>(a.out + (int64_t)row * a.hidden + col) = o;
}

// A work-group per 16 rows and 16 tokens; wave w takes the column blocks w, w + 8, ...
template <bool NORM>
__global__ __launch_bounds__(kW4Waves * 64) void w4_project_kernel(W4ProjectArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quarter = lane >> 4;
    const int tile = blockIdx.x, token = blockIdx.y * kW4Tokens + col;
    const int blocks = w4_blocks(a.hidden), groups = w4_groups(a.hidden, a.group);
    const int steps_per_group = a.group / 32;
    const bool there = token < a.n_tokens;
    const uint16_t* const x = a.x + (size_t)(there ? token : 0) * a.hidden;
    const u32x4* const w = reinterpret_cast<const u32x4*>(a.w) + (size_t)tile * blocks * 64 + lane;
    const uint2* const scales = reinterpret_cast<const uint2*>(a.scales) + ((size_t)tile * groups) * 4 + quarter;
    const u32x4 offset = {0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u};  // bf16 -136
    f32x4 y = {0.f, 0.f, 0.f, 0.f};  // rows 4 quarter + i, token `col`
    float squares = 0.f;
    for (int kb = wave; kb < blocks; kb += kW4Waves) {
        const u32x4 codes = __builtin_nontemporal_load(w + (size_t)kb * 64);
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = kb * 128 + 32 * s + 8 * quarter;
            u32x4 xb = {0u, 0u, 0u, 0u};
            if (there && k < a.hidden) {
                xb = *reinterpret_cast<const u32x4*>(x + k);
                if constexpr (NORM) {
                    const u32x4 g = *reinterpret_cast<const u32x4*>(a.gamma + k);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float lo = __uint_as_float(xb[j] << 16), hi = __uint_as_float(xb[j] & 0xFFFF0000u);
                        squares = fmaf(lo, lo, squares);
                        squares = fmaf(hi, hi, squares);
                        const bf16x2_t pair = {(__bf16)(lo * __uint_as_float(g[j] << 16)),
                                               (__bf16)(hi * __uint_as_float(g[j] & 0xFFFF0000u))};
                        xb[j] = __builtin_bit_cast(uint32_t, pair);
                    }
                }
            }
            u32x4 wa;
#pragma unroll
            for (int j = 0; j < 4; ++j) wa[j] = ((codes[s] >> (4 * j)) & 0x000F000Fu) | 0x43004300u;
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, wa), __builtin_bit_cast(bf16x8_t, xb), acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, offset), __builtin_bit_cast(bf16x8_t, xb), acc, 0, 0, 0);
            if ((s + 1) % steps_per_group == 0) {
                const uint2 four = scales[(size_t)((kb * 4 + s) / steps_per_group) * 4];
                y[0] = fmaf(__uint_as_float(four.x << 16), acc[0], y[0]);
                y[1] = fmaf(__uint_as_float(four.x & 0xFFFF0000u), acc[1], y[1]);
                y[2] = fmaf(__uint_as_float(four.y << 16), acc[2], y[2]);
                y[3] = fmaf(__uint_as_float(four.y & 0xFFFF0000u), acc[3], y[3]);
                acc = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
    __shared__ float part[kW4Waves][kW4Tokens][17];
    __shared__ float sums[kW4Waves][kW4Tokens];
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][col][4 * quarter + i] = y[i];
    if constexpr (NORM) {
        const float all = pair_sum32(pair_sum16(squares));
        if (quarter == 0) sums[wave][col] = all;
    }
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int t = threadIdx.x >> 4, r = threadIdx.x & 15;
    if (blockIdx.y * kW4Tokens + t >= a.n_tokens || tile * 16 + r >= a.rows) return;
    float out = 0.f;
#pragma unroll
    for (int i = 0; i < kW4Waves; ++i) out += part[i][t][r];
    if constexpr (NORM) {
        float total = 0.f;
#pragma unroll
        for (int i = 0; i < kW4Waves; ++i) total += sums[i][t];
        out *= 1.0f / sqrtf(total / (float)a.hidden + a.eps);
    }
    a.y[(size_t)(blockIdx.y * kW4Tokens + t) * a.ldy + tile * 16 + r] = __builtin_bit_cast(uint16_t, (__bf16)out);
}

}  // namespace

int64_t w4_packed_bytes(int rows, int hidden) { return (int64_t)((rows + 15) / 16) * w4_blocks(hidden) * 1024; }
int64_t w4_scale_bytes(int rows, int hidden, int group) { return (int64_t)((rows + 15) / 16) * w4_groups(hidden, group) * 32; }

static dim3 w4_grid(int rows, int hidden) {
    return dim3((uint32_t)((w4_packed_bytes(rows, hidden) / 4 + kW4Threads - 1) / kW4Threads));
}
hipError_t launch_w4_pack(const W4PackArgs& a, const Launch& l) {
    return launch_kernel(w4_pack_kernel, w4_grid(a.rows, a.hidden), dim3(kW4Threads), l, a);
}
hipError_t launch_w4_unpack(const W4UnpackArgs& a, const Launch& l) {
    return launch_kernel(w4_unpack_kernel, w4_grid(a.rows, a.hidden), dim3(kW4Threads), l, a);
}
hipError_t launch_w4_project(const W4ProjectArgs& a, const Launch& l) {
    const dim3 grid((a.rows + 15) / 16, (a.n_tokens + kW4Tokens - 1) / kW4Tokens), block(kW4Waves * 64);
    return a.gamma != nullptr ? launch_kernel(w4_project_kernel<true>, grid, block, l, a)
                              : launch_kernel(w4_project_kernel<false>, grid, block, l, a);
}

}  // namespace lara
