// Products with 4-bit weights: y[t, r] = inv_t * sum_g s[r, g] * sum_{k in g} (c[r, k] - 8) * (x[t, k] * gamma[k]), codes c of
// 0 .. 15, one bf16 scale per row r and group g of 32, 64 or 128 columns, inv_t = 1 / sqrt(mean(x_t^2) + eps) with gamma
// and 1 without.
//
// Packed form (gqa_w4_pack_device; a program packs its weights once): tiles of 16 rows x 128 columns, 1 KiB each, a row
// tile's column blocks in order.  Lane l of a wave owns 16 bytes of a tile: row l % 16, and in dword s its 8 columns
// 32s + 8 (l / 16) .. of the block: nibble j of the dword's low half is column 2j, of its high half 2j + 1.  So a wave
// reads a tile as 1 KiB in a row, dword s is operand A of one v_mfma_f32_16x16x32_bf16 whose 32 columns lie in one group
// (of any size), and (dword >> 4j) & 0x000F000F | 0x43004300 is a pair of bf16 128 + c.  Scales: [row tile][column
// block][4 rows'][group of the block][4], the order in which a lane reads them in one load or two.
// Rows past the matrix have code 8 and scale 0, columns past it scale 0.
//
// The constant 136 = 128 + 8 leaves through a product of its own, with operand A = -136 everywhere: it is the same for
// all rows, and a group's accumulators of every row tile start from it.  Products are exact and summed in fp32, a group at a
// time, then scaled in fp32.  x * gamma is rounded to bf16 (operand B; half a step of 2^-8, as the normalised rows of the bf16 stage are).
#include "gqa_internal.h"

#include <math.h>

namespace lara {
namespace {

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kW4Threads = 256;
constexpr int kW4Waves = 8;

__host__ __device__ inline int w4_blocks(int hidden) { return (hidden + 127) / 128; }
__host__ __device__ inline int w4_groups(int hidden, int group) { return w4_blocks(hidden) * (128 / group); }

// codes [rows][hidden / 2] (the even column in the low half of a byte), scales [rows][hidden / group] bf16.
__global__ __launch_bounds__(kW4Threads) void w4_pack_kernel(W4PackArgs a) {
    const int64_t i = (int64_t)wide_block() * kW4Threads + threadIdx.x;  // a dword of the packed codes
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
        const int per_block = 128 / a.group;
        const int64_t tile = i / (groups * 16);
        const int in = (int)(i % (groups * 16)), block = in / (16 * per_block), at = in % (16 * per_block);
        const int g = block * per_block + at / 4 % per_block, row = (int)tile * 16 + at / (4 * per_block) * 4 + at % 4;
        a.packed_scales[i] = row < a.rows && g < given ? a.scales[(int64_t)row * given + g] : (uint16_t)0;
    }
}

// The packed matrix as bf16 [rows][hidden]: (c - 8) * s, one rounding.
__global__ __launch_bounds__(kW4Threads) void w4_unpack_kernel(W4UnpackArgs a) {
    const int64_t i = (int64_t)wide_block() * kW4Threads + threadIdx.x;
    const int blocks = w4_blocks(a.hidden), tiles = (a.rows + 15) / 16;
    if (i >= (int64_t)tiles * blocks * 256) return;
    const int s = (int)(i & 3), lane = (int)(i >> 2) & 63;
    const int64_t tile = i >> 8;
    const int row_tile = (int)(tile / blocks), row = row_tile * 16 + (lane & 15);
    const int col = (int)(tile % blocks) * 128 + 32 * s + 8 * (lane >> 4);
    if (row >= a.rows || col >= a.hidden) return;
    const uint32_t c = a.packed[i];
    const int per_block = 128 / a.group;
    const float scale = __uint_as_float(
        (uint32_t)a.packed_scales[(tile * 4 + (lane >> 2 & 3)) * per_block * 4 + col % 128 / a.group * 4 + (lane & 3)] << 16);
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float even = (float)((int)((c >> (4 * j)) & 15u) - 8) * scale, odd = (float)((int)((c >> (16 + 4 * j)) & 15u) - 8) * scale;
        const bf16x2_t pair = {(__bf16)even, (__bf16)odd};
        o[j] = __builtin_bit_cast(uint32_t, pair);
    }
    *reinterpret_cast<u32x4*>(a.out + (int64_t)row * a.hidden + col) = o;
}

// Four rows of a token's y (those inside the matrix).
__device__ __forceinline__ void w4_store(const W4ProjectArgs& a, const f32x4& sum, int row, int token) {
    uint16_t* const to = a.y + (size_t)token * a.ldy + row;
    const bf16x2_t lo = {(__bf16)sum[0], (__bf16)sum[1]}, hi = {(__bf16)sum[2], (__bf16)sum[3]};
    const uint2 out = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
    if (row + 4 <= a.rows && (reinterpret_cast<uintptr_t>(to) & 7) == 0) {
        *reinterpret_cast<uint2*>(to) = out;
    } else {
        const uint16_t words[4] = {(uint16_t)out.x, (uint16_t)(out.x >> 16), (uint16_t)out.y, (uint16_t)(out.y >> 16)};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (row + i < a.rows) to[i] = words[i];
    }
}

// y += the four rows' scales * sum.
__device__ __forceinline__ void w4_add(f32x4& y, const uint2& scales, const f32x4& sum) {
    y[0] = fmaf(__uint_as_float(scales.x << 16), sum[0], y[0]);
    y[1] = fmaf(__uint_as_float(scales.x & 0xFFFF0000u), sum[1], y[1]);
    y[2] = fmaf(__uint_as_float(scales.y << 16), sum[2], y[2]);
    y[3] = fmaf(__uint_as_float(scales.y & 0xFFFF0000u), sum[3], y[3]);
}

// x + x of the lane that DPP control CTRL names.
template <int CTRL>
__device__ __forceinline__ float w4_row_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}

// 16 * NT tokens and RT row tiles a work-group of eight waves, which split the columns: wave w takes the blocks w, w + 8,
// ..., and its parts of y meet the others' in LDS at the end.  (Rows would not split: a launch of few tokens is the
// weights' latency, and only a split of the columns keeps every CU's share of them in flight at once.)
//
// A block's turn: the tokens' columns, loaded a turn ahead as whole lines (a lane has 8 columns of every fourth token), take
// gamma and go to LDS as operand B; nobody else reads these columns, so no barrier.  Straight from memory, operand B
// would be 16 rows at a stride a load and gamma the same 4 loads again, each multiplied in all 16 columns however few
// tokens there are: 13 tokens x 4096 -> 6144 took 10.5 us for 8.8, one token 9.1 for 7.0.  Codes and scales come
// straight from memory, also a turn ahead.  (Tokens that stay in LDS for the whole launch, work-groups going from tile to
// tile: 6.9 us for one token, 14.4 for 13, where every work-group's copy of the tokens is what it waits for.)
//
// What bounds it: at one token the weights' latency (4096 -> 6144, group 128, 13 MB: 7.0 us alone, 4.0 with other launches
// beside it, of which about 2.7 are the launch; 1.9 us at the read rate).  From 16 tokens on the unpacking of codes (7
// vector instructions for 8 codes a lane, used for 16 NT tokens) and the tokens' own way to every work-group.
//
// A token's sum is the same in every form: each wave adds its groups in order, the waves are added in order.
template <int NT, int RT, int SPG, bool NORM>
__global__ __launch_bounds__(kW4Waves * 64, NT * RT <= 2 && SPG == 4 ? 4 : 2) void w4_project_kernel(W4ProjectArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quarter = lane >> 4;
    const int blocks = w4_blocks(a.hidden), tiles = (a.rows + 15) / 16;
    const int tile0 = blockIdx.x * RT, token0 = blockIdx.y * 16 * NT;
    const int tokens = a.n_tokens - token0 < 16 * NT ? a.n_tokens - token0 : 16 * NT;
    constexpr int GROUPS = 4 / SPG;
    // A wave's own: its tokens' columns of a block (16 chunks of 8 and one of padding), in the end its part of y.
    constexpr int kXRow = 17, kLds = NT * (16 * kXRow > 64 * RT ? 16 * kXRow : 64 * RT);
    __shared__ u32x4 lds[kW4Waves][kLds];
    __shared__ float sums[kW4Waves][16 * NT];
    u32x4* const xw = lds[wave] + quarter * kXRow + col;
    const u32x4* const xr = lds[wave] + col * kXRow + quarter;
    struct Block {
        u32x4 codes[RT];
        uint2 scales[RT][GROUPS];
    };
    struct Tokens {
        u32x4 x[4 * NT], gamma;
    };
    const u32x4* w[RT];
    const uint16_t* scales[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {  // (a tile past the last: the last one, not written)
        const size_t tile = tile0 + r < tiles ? tile0 + r : tiles - 1;
        w[r] = reinterpret_cast<const u32x4*>(a.w) + tile * blocks * 64;
        scales[r] = a.scales + tile * blocks * GROUPS * 16;
    }
    const uint16_t* const x0 = a.x + (size_t)token0 * a.hidden;
    uint32_t x[4 * NT];  // tokens 4u + quarter (past the last: the last one, not written)
#pragma unroll
    for (int u = 0; u < 4 * NT; ++u) {
        const int token = 4 * u + quarter;
        x[u] = (uint32_t)(token < tokens ? token : tokens - 1) * a.hidden;
    }
    // Blocks past the last are the last one again, not used; for columns past the matrix stand the first (scale 0).
    auto load_x = [&](Tokens& b, int i) __attribute__((always_inline)) {
        const int kb = wave + kW4Waves * i, k = (kb < blocks ? kb : blocks - 1) * 128 + 8 * col, from = k < a.hidden ? k : 0;
#pragma unroll
        for (int u = 0; u < 4 * NT; ++u)
            if (4 * u < tokens) b.x[u] = *reinterpret_cast<const u32x4*>(x0 + (x[u] + from));
        if constexpr (NORM) b.gamma = *reinterpret_cast<const u32x4*>(a.gamma + from);
    };
    auto load = [&](Block& b, int i) __attribute__((always_inline)) {
        const int kb = wave + kW4Waves * i, in = kb < blocks ? kb : blocks - 1;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            b.codes[r] = __builtin_nontemporal_load(w[r] + (in * 64 + lane));
            const uint16_t* const s = scales[r] + (in * 4 + quarter) * GROUPS * 4;
            if constexpr (GROUPS == 1) {
                b.scales[r][0] = *reinterpret_cast<const uint2*>(s);
            } else {
#pragma unroll
                for (int g = 0; g < GROUPS; g += 2) {
                    const u32x4 two = *reinterpret_cast<const u32x4*>(s + 4 * g);
                    b.scales[r][g] = make_uint2(two[0], two[1]);
                    b.scales[r][g + 1] = make_uint2(two[2], two[3]);
                }
            }
        }
    };
    f32x4 y[RT][NT] = {};  // rows 4 quarter + i of tile r, token `col` of tile t
    float squares[4 * NT] = {};
    const u32x4 offset = {0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u};  // bf16 -136
    uint32_t bias = 0x43004300u;
    asm volatile("" : "+v"(bias));  // (in a register: v_and_or_b32 takes no constant)
    auto stage = [&](const Tokens& b, int i) __attribute__((always_inline)) {
        const int kb = wave + kW4Waves * i;
        if (kb >= blocks) return;
        const bool inside = kb * 128 + 8 * col < a.hidden;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int u = 0; u < 4 * NT; ++u) {
            if (4 * u >= tokens) break;
            u32x4 v = b.x[u];
            if constexpr (NORM) {
                float sum = squares[u];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bf16x2_t two = __builtin_bit_cast(bf16x2_t, (uint32_t)v[j]);
                    sum = __builtin_amdgcn_fdot2_f32_bf16(two, two, sum, false);
                    const float lo = __uint_as_float(v[j] << 16), hi = __uint_as_float(v[j] & 0xFFFF0000u);
                    const bf16x2_t pair = {(__bf16)(lo * __uint_as_float(b.gamma[j] << 16)),
                                           (__bf16)(hi * __uint_as_float(b.gamma[j] & 0xFFFF0000u))};
                    v[j] = __builtin_bit_cast(uint32_t, pair);
                }
                squares[u] = inside ? sum : squares[u];
            }
            xw[4 * u * kXRow] = v;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };
    auto product = [&](const Block& b, int i) __attribute__((always_inline)) {
        if (wave + kW4Waves * i >= blocks) return;
        f32x4 acc[RT][NT];
#pragma unroll
        for (int s0 = 0; s0 < 4; s0 += SPG) {
            bf16x8_t xb[SPG][NT];
#pragma unroll
            for (int s = 0; s < SPG; ++s)
#pragma unroll
                for (int t = 0; t < NT; ++t) xb[s][t] = __builtin_bit_cast(bf16x8_t, xr[16 * t * kXRow + 4 * (s0 + s)]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4 all = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = s0; s < s0 + SPG; ++s)
                    all = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, offset), xb[s - s0][t], all, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[r][t] = all;
            }
#pragma unroll
            for (int s = s0; s < s0 + SPG; ++s)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    u32x4 wa;
#pragma unroll
                    for (int j = 0; j < 4; ++j) wa[j] = ((b.codes[r][s] >> (4 * j)) & 0x000F000Fu) | bias;
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        acc[r][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, wa), xb[s - s0][t], acc[r][t], 0, 0, 0);
                }
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int t = 0; t < NT; ++t) w4_add(y[r][t], b.scales[r][s0 / SPG], acc[r][t]);
        }
    };
    // (32 tokens' columns are held once, for registers: the next are loaded when these are in LDS.)
    constexpr bool kTwice = NT == 1;
    Block block[2];
    Tokens xs[kTwice ? 2 : 1];
    load_x(xs[0], 0);
    load(block[0], 0);
    const int turns = (blocks + kW4Waves - 1) / kW4Waves;
    auto turn = [&](int i, const Block& now, Block& next, Tokens& x_now, Tokens& x_next) __attribute__((always_inline)) {
        if constexpr (kTwice) load_x(x_next, i + 1);
        load(next, i + 1);
        stage(x_now, i);
        if constexpr (!kTwice) load_x(x_next, i + 1);
        product(now, i);
    };
    for (int i = 0; i < turns; i += 2) {
        turn(i, block[0], block[1], xs[0], xs[kTwice ? 1 : 0]);
        if (i + 1 < turns) turn(i + 1, block[1], block[0], xs[kTwice ? 1 : 0], xs[0]);
    }
    if constexpr (NORM) {
#pragma unroll
        for (int u = 0; u < 4 * NT; ++u) {
            float v = w4_row_add<0x128>(squares[u]);  // row_ror 8, 4, 2, 1
            v = w4_row_add<0x124>(v);
            v = w4_row_add<0x122>(v);
            v = w4_row_add<0x121>(v);
            if (col == 0) sums[wave][4 * u + quarter] = v;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) lds[wave][(r * NT + t) * 64 + lane] = __builtin_bit_cast(u32x4, y[r][t]);
    __syncthreads();
    for (int p = wave; p < RT * NT; p += kW4Waves) {
        const int r = p / NT, t = p - r * NT, token = 16 * t + col;
        f32x4 sum = __builtin_bit_cast(f32x4, lds[0][p * 64 + lane]);
#pragma unroll
        for (int i = 1; i < kW4Waves; ++i) sum += __builtin_bit_cast(f32x4, lds[i][p * 64 + lane]);
        if constexpr (NORM) {
            float total = 0.f;
#pragma unroll
            for (int i = 0; i < kW4Waves; ++i) total += sums[i][token];
            sum *= 1.0f / sqrtf(total / (float)a.hidden + a.eps);
        }
        if (token < tokens) w4_store(a, sum, (tile0 + r) * 16 + 4 * quarter, token0 + token);
    }
}

}  // namespace

int64_t w4_packed_bytes(int rows, int hidden) { return (int64_t)((rows + 15) / 16) * w4_blocks(hidden) * 1024; }
int64_t w4_scale_bytes(int rows, int hidden, int group) { return (int64_t)((rows + 15) / 16) * w4_groups(hidden, group) * 32; }

static dim3 w4_grid(int rows, int hidden) {
    return wide_grid((w4_packed_bytes(rows, hidden) / 4 + kW4Threads - 1) / kW4Threads);
}
hipError_t launch_w4_pack(const W4PackArgs& a, const Launch& l) {
    return launch_kernel(w4_pack_kernel, w4_grid(a.rows, a.hidden), dim3(kW4Threads), l, a);
}
hipError_t launch_w4_unpack(const W4UnpackArgs& a, const Launch& l) {
    return launch_kernel(w4_unpack_kernel, w4_grid(a.rows, a.hidden), dim3(kW4Threads), l, a);
}
namespace {
template <int NT, int RT, int SPG>
hipError_t w4_launch(const W4ProjectArgs& a, const Launch& l) {
    const dim3 grid(((a.rows + 15) / 16 + RT - 1) / RT, (a.n_tokens + 16 * NT - 1) / (16 * NT)), block(kW4Waves * 64);
    return a.gamma != nullptr ? launch_kernel(w4_project_kernel<NT, RT, SPG, true>, grid, block, l, a)
                              : launch_kernel(w4_project_kernel<NT, RT, SPG, false>, grid, block, l, a);
}

template <int NT, int RT>
hipError_t w4_launch(const W4ProjectArgs& a, const Launch& l) {
    return a.group == 32 ? w4_launch<NT, RT, 1>(a, l) : a.group == 64 ? w4_launch<NT, RT, 2>(a, l) : w4_launch<NT, RT, 4>(a, l);
}
}  // namespace

// More rows and tokens a work-group: fewer copies of the tokens and codes unpacked once for more of them, but fewer
// work-groups; the largest form that leaves 5 / 8 of the CUs one.  Alone, us, 1 / 2 / 4 row tiles of 16 tokens, 4 of
// 32: 1 token 4096 -> 6144 7.5 / 6.6 / 8.6 (384 / 192 / 96 work-groups); 5 tokens 2080 -> 1000 4.6 / 5.5 / 7.4 (63 and less);
// 8 tokens 8192 -> 10240 20.0 / 20.8 / 15.4 (640 / 320 / 160); 64 tokens 2048 -> 4096 9.2 / 8.0 / 6.7 / 8.3 (the last two:
// 256, 128); 40 tokens 4096 -> 6144 21.0 / 19.1 / 16.9 / 13.4 (288, 192).
hipError_t launch_w4_project(const W4ProjectArgs& a, int n_cu, const Launch& l) {
    const int64_t tiles = (a.rows + 15) / 16, of16 = (a.n_tokens + 15) / 16, of32 = (a.n_tokens + 31) / 32;
    const int64_t enough = (5 * (int64_t)n_cu + 7) / 8;
    if (a.n_tokens > 16 && (tiles + 3) / 4 * of32 >= enough) return w4_launch<2, 4>(a, l);
    if ((tiles + 3) / 4 * of16 >= enough) return w4_launch<1, 4>(a, l);
    if ((tiles + 1) / 2 * of16 >= enough) return w4_launch<1, 2>(a, l);
    return w4_launch<1, 1>(a, l);
}

}  // namespace lara
