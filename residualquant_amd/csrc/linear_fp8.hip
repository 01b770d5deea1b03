// Projections in 8-bit floating point: with E4M3 codes c and block scales s,
//   y[m, n] = bf16(sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} cx[m, k] cw[n, k]),
// blocks of 128 inputs.  sx[m, b] is the least power of two >= 2^-126 with
// |x| <= 448 sx for the block's finite values, cx = x / sx to nearest, ties to
// even; sw is given for 128 outputs x 128 inputs, as an exponent (E8M0) or in FP32.
//
// Both operands lie in tiles of 16 rows x 128 inputs, 2 KB each, in the order in
// which v_mfma_scale_f32_16x16x128 takes them: lane l = (i = l % 16, g = l / 16)
// holds row i, inputs 8 g.. and 32 + 8 g.. (eight each) in the 16 bytes at 16 l, 64 +
// 8 g.. and 96 + 8 g.. at 1024 + 16 l.  (An instruction sums over all 128 inputs, so
// their order matters only in that both operands have the same; in this one, four
// lanes together read 64 bytes of a BF16 row at a time.)  Rows and inputs past the matrix
// hold 0.
// Of 32 outputs, tile t (0, 1) holds the outputs 8 g + 4 t + r as its rows 4 g + r: a
// lane of the result, which has rows 4 g + 0..3 of a tile, then has 8 neighbouring
// outputs of both tiles, and a row's 32 outputs are stored as 64 bytes at once.
// Weights lie as [64 outputs][block][tile][2 KB], x as [block][tile][2 KB]: what the
// waves read at a time is whole stretches of 8 KB and more, which all channels of
// the L2 cache hold alike.  (With each tile's blocks in a row, at 2048 inputs a tile
// begins every 32 KB, and workgroups at the same block met in half the channels.)
// The instruction multiplies by powers of two as it goes: sx and sw, if that is an
// exponent. An FP32 sw is split in two: its power of two goes the same way and the factor of [1, 2)
// that is left multiplies the block's FP32 sum, so that this is in range wherever the
// block's part of the result is. (With sw multiplied afterwards, scales of 2^-12 and results
// from 2^116 on, the sum before passed 2^128.)
//
// What the 8-bit instructions cost in exactness: beside FP32 sums they line the 16
// products of a lane's piece up with the largest and cut what lies below 2^-13 of its power of two.
// Against sums in 64 bits results are off by 1.4e-5 (normal values) to 5.6e-5 (codes of
// all sizes) in the 2-norm, at 128 as at 2048 inputs, a hundredth of what the
// rounding to BF16 is off by (1.7e-3). v_mfma_f32_16x16x32_fp8_fp8 cuts alike;
// codes converted to BF16 operands would not (3e-7), at half the rate and with a
// conversion per two codes.
#include <algorithm>
#include <type_traits>

#include "rq_device.h"
#include "rq_fp8.h"
#include "rq_reduced.h"

namespace rq {

namespace {

typedef float F32x4 __attribute__((ext_vector_type(4)));
typedef int I32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = 128, kTileBytes = 16 * kBlock;

// Behind x's codes and scales in the workspace: what the wide kernels read past the last row tile, of the
// codes up to seven tiles.
constexpr int kPastRows = 8 * kTileBytes;

// Results at any element (rows of an odd number of outputs begin at any).
typedef U32x4 U32x4At2 __attribute__((aligned(2)));
typedef U32x2 U32x2At2 __attribute__((aligned(2)));

// The input of byte e (0..15) of lane group g's piece `half`, within its block.
__device__ __forceinline__ int input_of(int half, int g, int e) { return 64 * half + 32 * (e >> 3) + 8 * g + (e & 7); }

__host__ __device__ __forceinline__ int64_t tiles_of(int64_t rows) { return (rows + 15) / 16; }
// (Whole groups of 64, as the waves of the product for many rows take them.)
__host__ __device__ __forceinline__ int64_t out_tiles_of(int64_t out_features) { return (out_features + 63) / 64 * 4; }
// The output that row `row` of a tile stands for.
__device__ __forceinline__ int64_t output_of(int64_t tile, int row) {
    return 32 * (tile >> 1) + 8 * (row >> 2) + 4 * (int)(tile & 1) + (row & 3);
}
// Places of a weight's tile and of a tile of x, in tiles.
__device__ __forceinline__ int64_t weight_place(int64_t tile, int64_t blocks, int64_t block) {
    return 4 * ((tile >> 2) * blocks + block) + (tile & 3);
}
__device__ __forceinline__ int64_t row_place(int64_t tile, int64_t row_tiles, int64_t block) { return block * row_tiles + tile; }

__host__ __device__ __forceinline__ int64_t blocks_of(int64_t in_features) { return (in_features + kBlock - 1) / kBlock; }
// Scales lie in fours, one word per row (or block row) and four blocks.
__host__ __device__ __forceinline__ int64_t fours_of(int64_t in_features) { return (blocks_of(in_features) + 3) / 4; }

// The exponent byte (E8M0, 2^(byte - 127)) of a block's scale.
__device__ __forceinline__ int scale_exponent(float largest) { return (int)(__float_as_uint(needed_scale(largest)) >> 23); }
// 2^(127 - byte): what a value is multiplied by before its rounding, exactly (byte <= 247).
__device__ __forceinline__ float inverse_scale(int exponent) { return __uint_as_float((uint32_t)(254 - exponent) << 23); }

// An FP32 scale as 2^(power - 127) x factor, exactly: |factor| in [1, 2), below for a subnormal scale; what is
// not finite stays in the factor.
__device__ __forceinline__ uint32_t scale_power(float scale) {
    return min(max((__float_as_uint(scale) >> 23) & 0xffu, 1u), 254u);
}
__device__ __forceinline__ float scale_factor(float scale, uint32_t power) { return __builtin_amdgcn_ldexpf(scale, 127 - (int)power); }

__device__ __forceinline__ float finite_size(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.f; }

// ------------------------------------------------------------------ weights

// One thread per 16 bytes of the packed codes.
__global__ __launch_bounds__(256) void pack_fp8_kernel(const Fp8PackParams p) {
    const int64_t blocks = blocks_of(p.in_features), pieces = out_tiles_of(p.out_features) * blocks * (kTileBytes / 16);
    const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t high = (p.out_features + kBlock - 1) / kBlock, wide = 4 * fours_of(p.in_features);
    if (w < high * wide) {
        const int64_t row = w / wide, block = w % wide, from = row * blocks + block;
        if (p.exponents)
            p.packed_scales[w] = block < blocks ? static_cast<const uint8_t*>(p.scales)[from] : 127;
        else
            reinterpret_cast<float*>(p.packed_scales)[w] = block < blocks ? static_cast<const float*>(p.scales)[from] : 0.f;
    }
    if (w >= pieces) return;
    const int lane = (int)w & 63, half = (int)(w >> 6) & 1;
    const int64_t block = (w >> 9) % blocks, n = output_of(4 * ((w >> 9) / blocks) + ((w >> 7) & 3), lane & 15);
    U32x4 piece = {0u, 0u, 0u, 0u};
    if (n < p.out_features)
        for (int e = 0; e < 16; ++e) {
            const int64_t k = kBlock * block + input_of(half, lane >> 4, e);
            if (k < p.in_features) piece[e >> 2] |= (uint32_t)p.codes[n * p.in_features + k] << (8 * (e & 3));
        }
    reinterpret_cast<U32x4*>(p.packed)[w] = piece;
}

// One workgroup per block of 128 outputs x 128 inputs of a BF16 weight.
__global__ __launch_bounds__(256) void quantize_weight_fp8_kernel(const Fp8PackParams p) {
    __shared__ float largest_of[4];
    const int64_t blocks = blocks_of(p.in_features), block = blockIdx.x % blocks, high = blockIdx.x / blocks;
    float largest = 0.f;
    for (int e = threadIdx.x; e < kBlock * kBlock; e += 256) {
        const int64_t n = kBlock * high + e / kBlock, k = kBlock * block + e % kBlock;
        if (n < p.out_features && k < p.in_features) largest = fmaxf(largest, finite_size(bf16_f32(p.weight[n * p.in_features + k])));
    }
    for (int d = 32; d; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
    if ((threadIdx.x & 63) == 0) largest_of[threadIdx.x >> 6] = largest;
    __syncthreads();
    for (int w = 0; w < 4; ++w) largest = fmaxf(largest, largest_of[w]);
    const int exponent = scale_exponent(largest);
    const int64_t wide = 4 * fours_of(p.in_features);
    if (threadIdx.x == 0) {
        p.packed_scales[high * wide + block] = (uint8_t)exponent;
        if (block == blocks - 1)
            for (int64_t b = blocks; b < wide; ++b) p.packed_scales[high * wide + b] = 127;
    }
    const float inverse = inverse_scale(exponent);
    const int64_t tiles = out_tiles_of(p.out_features);
    for (int w = threadIdx.x; w < 8 * (kTileBytes / 16); w += 256) {
        const int lane = w & 63, half = (w >> 6) & 1;
        const int64_t tile = 8 * high + (w >> 7), n = output_of(tile, lane & 15);
        if (tile >= tiles) continue;
        float x[16];
        for (int e = 0; e < 16; ++e) {
            const int64_t k = kBlock * block + input_of(half, lane >> 4, e);
            x[e] = n < p.out_features && k < p.in_features ? bf16_f32(p.weight[n * p.in_features + k]) * inverse : 0.f;
        }
        U32x4 piece;
        for (int e = 0; e < 4; ++e) piece[e] = fp8x4_rn(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        reinterpret_cast<U32x4*>(p.packed)[(weight_place(tile, blocks, block) * 2 + half) * 64 + lane] = piece;
    }
}

// The BF16 weight [out, in] of a packed one: bf16(code x scale).  One thread per 16 bytes.
__global__ __launch_bounds__(256) void unpack_fp8_kernel(const Fp8PackParams p, uint16_t* weight) {
    const int64_t blocks = blocks_of(p.in_features), pieces = out_tiles_of(p.out_features) * blocks * (kTileBytes / 16);
    const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (w >= pieces) return;
    const int lane = (int)w & 63, half = (int)(w >> 6) & 1;
    const int64_t block = (w >> 9) % blocks, n = output_of(4 * ((w >> 9) / blocks) + ((w >> 7) & 3), lane & 15);
    if (n >= p.out_features) return;
    const int64_t at = n / kBlock * (4 * fours_of(p.in_features)) + block;
    float scale;
    if (p.exponents) {
        const uint32_t e = p.packed_scales[at];
        scale = e == 255 ? __builtin_nanf("") : e == 0 ? 0x1p-127f : __uint_as_float(e << 23);
    } else {
        scale = reinterpret_cast<const float*>(p.packed_scales)[at];
    }
    const U32x4 piece = reinterpret_cast<const U32x4*>(p.packed)[w];
    for (int e = 0; e < 16; ++e) {
        const int64_t k = kBlock * block + input_of(half, lane >> 4, e);
        if (k < p.in_features) weight[n * p.in_features + k] = (uint16_t)bf16_rn(e4m3_f32((piece[e >> 2] >> (8 * (e & 3))) & 0xffu) * scale);
    }
}

// ------------------------------------------------------------------ rows

// Eight neighbouring values of a row of any alignment and length (0 past its end).
__device__ __forceinline__ U32x4 load_values(const uint16_t* row, int64_t k, int64_t in_features) {
    U32x4 raw;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        raw[e] = (k + 2 * e < in_features ? row[k + 2 * e] : 0u) | (k + 2 * e + 1 < in_features ? (uint32_t)row[k + 2 * e + 1] << 16 : 0u);
    return raw;
}

// A block of a row, 32 values in each of the lanes i, i + 16, i + 32, i + 48 of a wave: its scale, and these
// values' operands.
__device__ __forceinline__ float quantize_row_block(const U32x4 (&raw)[4], I32x8& codes) {
    auto largest_of = [&](bool finite) {
        uint32_t most = 0;
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) most = larger_sizes(most, finite ? finite_sizes(raw[h][e]) : raw[h][e] & 0x7fff7fffu);
        most = max(most >> 16, most & 0xffffu);
        most = max(most, (uint32_t)__shfl_xor((int)most, 16));
        return max(most, (uint32_t)__shfl_xor((int)most, 32));
    };
    uint32_t most = largest_of(false);
    if (__any(most >= kBf16Infinity)) most = largest_of(true);
    const float scale = needed_scale(__uint_as_float(most << 16));
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        codes[2 * h] = (int)fp8x4_of_bf16(raw[h][0], raw[h][1], scale);
        codes[2 * h + 1] = (int)fp8x4_of_bf16(raw[h][2], raw[h][3], scale);
    }
    return scale;
}

// One workgroup per tile of 16 rows and four blocks of 128 inputs, a wave a block: lane (i, g) the operands
// of row i, inputs 32 h + 8 g.. (eight each). Eights: whole pieces of eight inputs, read at any alignment and
// without a condition (16-byte loads that one path leaves out wait one by one).
template <bool Eights>
__global__ __launch_bounds__(256) void quantize_rows_fp8_kernel(const LinearFp8Params p) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
    const int64_t blocks = blocks_of(p.in_features), fours = fours_of(p.in_features), row_tiles = tiles_of(p.rows);
    const int64_t four = blockIdx.x % fours, tile = blockIdx.x / fours, m = 16 * tile + i, b = 4 * four + wave;
    const int64_t in_features = m < p.rows ? p.in_features : 0;
    const int64_t k = kBlock * b + 8 * g;
    U32x4 raw[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        if constexpr (Eights)
            raw[h] = *reinterpret_cast<const U32x4At2*>(p.x + (k + 32 * h < in_features ? m * p.x_stride + k + 32 * h : 0));
        else
            raw[h] = load_values(p.x + m * p.x_stride, k + 32 * h, in_features);
    }
    if constexpr (Eights)
#pragma unroll
        for (int h = 0; h < 4; ++h)
            if (k + 32 * h >= in_features) raw[h] = U32x4{0u, 0u, 0u, 0u};
    I32x8 codes;
    const float scale = quantize_row_block(raw, codes);
    if (b < blocks) {
        uint8_t* const to = p.x_codes + row_place(tile, row_tiles, b) * kTileBytes + 16 * lane;
        *reinterpret_cast<U32x4*>(to) = U32x4{(uint32_t)codes[0], (uint32_t)codes[1], (uint32_t)codes[2], (uint32_t)codes[3]};
        *reinterpret_cast<U32x4*>(to + 1024) = U32x4{(uint32_t)codes[4], (uint32_t)codes[5], (uint32_t)codes[6], (uint32_t)codes[7]};
    }
    if (g == 0) reinterpret_cast<uint8_t*>(p.x_scales)[4 * ((four * row_tiles + tile) * 16 + i) + wave] = (uint8_t)(__float_as_uint(scale) >> 23);
}

// ------------------------------------------------------------------ product

__device__ __forceinline__ I32x8 operand(const uint8_t* tile, int lane) {
    const U32x4 a = *reinterpret_cast<const U32x4*>(tile + 16 * lane), b = *reinterpret_cast<const U32x4*>(tile + 1024 + 16 * lane);
    return I32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// 16 outputs (a) x 16 rows (b) over 128 inputs; lane (i, g) of the result: row i, outputs 4 g + 0..3.
// The scales are bytes A and B of their words.
template <int A = 0, int B = 0>
__device__ __forceinline__ F32x4 mfma(I32x8 a, I32x8 b, F32x4 c, uint32_t scale_a, uint32_t scale_b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, A, (int)scale_a, B, (int)scale_b);
}

// Up to some hundred rows: one workgroup of eight waves per J tiles of outputs and T tiles of 16 rows. The
// waves share the inputs out, each with operands straight from global memory (whole
// stretches of 2 KB), two blocks in turn, and join through LDS.
template <int J, int T, bool Exponents>
__global__ __launch_bounds__(512) void linear_fp8_split_kernel(const LinearFp8Params p) {
    __shared__ F32x4 partial[8][J * T][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int blocks = (int)blocks_of(p.in_features), fours = (int)fours_of(p.in_features);
    const int64_t row_tiles = tiles_of(p.rows), row_groups = (row_tiles + T - 1) / T;
    const int64_t tile0 = J * (blockIdx.x / row_groups), row_tile0 = T * (blockIdx.x % row_groups);
    const int begin = blocks * wave / 8, end = blocks * (wave + 1) / 8;
    typedef std::conditional_t<Exponents, uint32_t, float> Scale;
    struct Block {
        I32x8 a[J], x[T];
        uint32_t words[T];
        Scale scale;
    };
    auto load = [&](Block& to, int b) {
#pragma unroll
        for (int j = 0; j < J; ++j) to.a[j] = operand(p.packed + weight_place(tile0 + j, blocks, b) * kTileBytes, lane);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int64_t m = min(row_tile0 + t, row_tiles - 1);
            to.x[t] = operand(p.x_codes + row_place(m, row_tiles, b) * kTileBytes, lane);
            to.words[t] = p.x_scales[((b >> 2) * row_tiles + m) * 16 + i];
        }
        if constexpr (Exponents)
            to.scale = reinterpret_cast<const uint32_t*>(p.packed_scales)[tile0 / 8 * fours + (b >> 2)];
        else
            to.scale = reinterpret_cast<const float*>(p.packed_scales)[tile0 / 8 * (4 * fours) + b];
    };
    F32x4 total[J][T];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int t = 0; t < T; ++t) total[j][t] = F32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Block& of, int b) {
        const int shift = 8 * (b & 3);
        uint32_t power = 0;
        float factor = 0.f;
        if constexpr (!Exponents) power = scale_power(of.scale), factor = scale_factor(of.scale, power);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int t = 0; t < T; ++t) {
                if constexpr (Exponents) {
                    total[j][t] = mfma(of.a[j], of.x[t], total[j][t], of.scale >> shift, of.words[t] >> shift);
                } else {
                    const F32x4 sum = mfma(of.a[j], of.x[t], F32x4{0.f, 0.f, 0.f, 0.f}, power, of.words[t] >> shift);
#pragma unroll
                    for (int r = 0; r < 4; ++r) total[j][t][r] = fmaf(factor, sum[r], total[j][t][r]);
                }
            }
    };
    // (Past the end the last block is loaded again. The compiler moves next's loads into the branch that multiplies it,
    // behind the loads of the block after it, and the wait there is for all of them: a pair of blocks pays one round
    // trip that no product covers.)
    Block now, next;
    load(now, min(begin, blocks - 1));
    for (int b = begin; b < end; b += 2) {
        load(next, min(b + 1, blocks - 1));
        multiply(now, b);
        load(now, min(b + 2, blocks - 1));
        if (b + 1 < end) multiply(next, b + 1);
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
        for (int t = 0; t < T; ++t) partial[wave][j * T + t][lane] = total[j][t];
    __syncthreads();
    // The waves share the tiles out, a pair with neighbouring outputs at a time.
    for (int q = wave; q < J / 2 * T; q += 8) {
        const int j = 2 * (q / T), t = q % T;
        F32x4 sum[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[h] = partial[0][(j + h) * T + t][lane];
#pragma unroll
            for (int w = 1; w < 8; ++w) sum[h] += partial[w][(j + h) * T + t][lane];
        }
        const int64_t n = output_of(tile0 + j, 4 * g), m = 16 * (row_tile0 + t) + i;
        if (m >= p.rows) continue;
        uint16_t* const to = p.y + m * p.y_stride + n;
        if (n + 8 <= p.out_features) {
            const F32x4 u = sum[0], v = sum[1];
            *reinterpret_cast<U32x4At2*>(to) = U32x4{bf16x2_rn(u[0], u[1]), bf16x2_rn(u[2], u[3]), bf16x2_rn(v[0], v[1]), bf16x2_rn(v[2], v[3])};
            continue;
        }
#pragma unroll
        for (int r = 0; r < 8; ++r)
            if (n + r < p.out_features) to[r] = (uint16_t)bf16_rn(r < 4 ? sum[0][r] : sum[1][r - 4]);
    }
}

// Few rows: one launch. Workgroups of W waves take tiles of 16 outputs one
// after the other, for all rows (T tiles of 16); the waves share the inputs out and
// join through LDS. A wave rounds its at most B blocks of x once, straight into operands
// that stay in its registers, while its first weights are on the way; a tile's weights are all asked
// for while the tile before it is joined. (x rounded into LDS by all waves: 8 rows, 2048 -> 6144
// 7.3 us, and 4.7 so.)
template <int T, int W, int B, bool Exponents>
__global__ __launch_bounds__(64 * W) void linear_fp8_few_kernel(const LinearFp8Params p) {
    __shared__ F32x4 partial[2][W][T][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4, rows = (int)p.rows;
    const int blocks = (int)blocks_of(p.in_features), fours = (int)fours_of(p.in_features);
    const int begin = blocks * wave / W, count = blocks * (wave + 1) / W - begin;
    const int64_t tiles = out_tiles_of(p.out_features);
    int64_t tile = blockIdx.x;
    typedef std::conditional_t<Exponents, uint32_t, float> Scale;
    struct Block {
        I32x8 a;
        Scale scale;
    };
    // (Loads without a condition, past the end the last block again: after a load that one path leaves out every wait
    // is for all loads in flight.)
    auto load = [&](Block& to, int b) {
        b = min(begin + b, blocks - 1);
        to.a = operand(p.packed + weight_place(tile, blocks, b) * kTileBytes, lane);
        if constexpr (Exponents)
            to.scale = p.packed_scales[tile / 8 * (4 * fours) + b];
        else
            to.scale = reinterpret_cast<const float*>(p.packed_scales)[tile / 8 * (4 * fours) + b];
    };
    Block held[B];
    // Lane (i, g): row i of a tile, inputs 32 h + 8 g.. of a block (eight each), h = 0..3.
    constexpr uint32_t kOutside = 1u << 31;  // past x's bytes, with what is added below too
    const int in_features = (int)p.in_features;
    const __amdgpu_buffer_rsrc_t x_all = handoff_resource(p.x, (uint32_t)((p.rows - 1) * p.x_stride + p.in_features) * 2);
    struct Raw {
        U32x4 piece[4];
    };
    auto load_raw = [&](int q) {
        const int b = q / T, row = 16 * (q % T) + i, k = kBlock * (begin + b) + 8 * g;
        // (What lies outside of x reads as 0.)
        const uint32_t at = row < rows && b < count ? (uint32_t)(row * p.x_stride + k) * 2 : kOutside;
        Raw raw;
        if (!p.wide) {
            const uint16_t* const from = p.x + row * p.x_stride;
#pragma unroll
            for (int h = 0; h < 4; ++h)
                raw.piece[h] = load_values(from, k + 32 * h, row < rows && b < count ? in_features : 0);
            return raw;
        }
#pragma unroll
        for (int h = 0; h < 4; ++h)
            raw.piece[h] = __builtin_amdgcn_raw_buffer_load_b128(x_all, k + 32 * h < in_features ? at + 64 * h : kOutside, 0, 0);
        return raw;
    };
    I32x8 x[B][T];
    uint32_t x_scales[(B * T + 3) / 4];  // four bytes each
    auto round = [&](const Raw& raw, int q) {
        const float scale = quantize_row_block(raw.piece, x[q / T][q % T]);
        if (q % 4 == 0) x_scales[q / 4] = 0;
        x_scales[q / 4] |= (__float_as_uint(scale) >> 23) << (8 * (q % 4));
    };
    // x, which lies in the L2 cache once the first workgroups have read it, is asked for first and rounded while the
    // weights are on the way: loads return in their order.
    constexpr int kFirst = B * T < 4 ? B * T : 4;
    Raw raw[kFirst];
#pragma unroll
    for (int q = 0; q < kFirst; ++q) raw[q] = load_raw(q);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int b = 0; b < B; ++b) load(held[b], b);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int q = 0; q < kFirst; ++q) round(raw[q], q);
#pragma unroll
    for (int q = kFirst; q < B * T; ++q) round(load_raw(q), q);
    int side = 0;
    while (true) {
        F32x4 total[T];
#pragma unroll
        for (int t = 0; t < T; ++t) total[t] = F32x4{0.f, 0.f, 0.f, 0.f};
        const int64_t own = tile;
        tile += gridDim.x;
        const bool more = tile < tiles;
        if (!more) tile = own;
        auto multiply = [&](auto place) {
            constexpr int Q = decltype(place)::value, b = Q / T, t = Q % T;
            if constexpr (Exponents) {
                total[t] = mfma<0, Q % 4>(held[b].a, x[b][t], total[t], held[b].scale, x_scales[Q / 4]);
            } else {
                const uint32_t power = scale_power(held[b].scale);
                const float factor = scale_factor(held[b].scale, power);
                const F32x4 sum = mfma<0, Q % 4>(held[b].a, x[b][t], F32x4{0.f, 0.f, 0.f, 0.f}, power, x_scales[Q / 4]);
#pragma unroll
                for (int r = 0; r < 4; ++r) total[t][r] = fmaf(factor, sum[r], total[t][r]);
            }
        };
        auto block = [&](auto number) {
            constexpr int b = decltype(number)::value;
            // (What lies past the wave's last block may hold NaN: no product of it, not even with 0.)
            if (b < count) {
                multiply(std::integral_constant<int, b * T>{});
                if constexpr (T > 1) multiply(std::integral_constant<int, b * T + 1>{});
                if constexpr (T > 2) multiply(std::integral_constant<int, b * T + 2>{});
            }
            load(held[b], b);  // the next tile's
        };
        block(std::integral_constant<int, 0>{});
        if constexpr (B > 1) block(std::integral_constant<int, 1>{});
        if constexpr (B > 2) block(std::integral_constant<int, 2>{});
        if constexpr (B > 3) block(std::integral_constant<int, 3>{});
#pragma unroll
        for (int t = 0; t < T; ++t) partial[side][wave][t][lane] = total[t];
        lds_barrier();
        if (wave < T) {
            const int t = wave;
            F32x4 sum = partial[side][0][t][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) sum += partial[side][w][t][lane];
            const int64_t n = output_of(own, 4 * g);
            const int row = 16 * t + i;
            if (row < rows) {
                uint16_t* const to = p.y + row * p.y_stride + n;
                if (n + 4 <= p.out_features) {
                    *reinterpret_cast<U32x2At2*>(to) = U32x2{bf16x2_rn(sum[0], sum[1]), bf16x2_rn(sum[2], sum[3])};
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n + r < p.out_features) to[r] = (uint16_t)bf16_rn(sum[r]);
                }
            }
        }
        if (!more) return;
        side ^= 1;  // (whose last readers passed the barrier above)
    }
}

// Many rows: workgroups of four waves take tiles of 256 outputs and 16 NT rows, a
// wave 64 outputs.  x passes LDS, where the four waves of its rows
// read it, in a ring of four blocks of inputs with a barrier every two; the weights
// go from global memory to the operands, since their order there is the operands'
// own and no two waves of a workgroup share them.  (Through LDS both would take it 128 bytes a
// cycle, all that it has, at the matrix instructions' full rate.)  What a block
// reads from global memory was asked for a block ahead, and a tile's first block
// before the results of the tile before it are stored.  (Two waits are for every load in
// flight: the next four blocks' scales are made uniform as soon as they are asked for, and a
// tile begins with the rows of two blocks loaded and stored in turn.)
template <bool Exponents, int NT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) void linear_fp8_wide_kernel(const LinearFp8Params p) {
    constexpr int kPieces = NT * kTileBytes / 16 / 256;  // 16-byte pieces of x per thread and block
    __shared__ __align__(16) uint8_t lds[4][NT * kTileBytes];
    __shared__ uint32_t x_words[2][16 * NT];  // scales of its rows, for four blocks each
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int blocks = (int)blocks_of(p.in_features), fours = (int)fours_of(p.in_features);
    const int64_t out_groups = (p.out_features + 255) / 256, row_groups = (p.rows + 16 * NT - 1) / (16 * NT);
    const int64_t out_tiles = out_tiles_of(p.out_features), row_tiles = tiles_of(p.rows);
    // (In 32 bits: rows_at_once.)
    const uint32_t x_stride = (uint32_t)row_tiles * kTileBytes, words_stride = (uint32_t)row_tiles * 64;

    // Neighbouring workgroups run on different XCDs: each XCD takes a stretch of the
    // tiles, eight row groups wide, whose weights and rows its workgroups share.
    const int64_t tiles = out_groups * row_groups, per = (tiles + 7) / 8;
    const int64_t stop = min(((int64_t)(blockIdx.x & 7) + 1) * per, tiles);
    const int step_of_tiles = gridDim.x >> 3;
    int64_t tile0, row_tile0;  // of this wave's outputs, of the rows
    __amdgpu_buffer_rsrc_t weights, x_all, x_scales;
    typedef std::conditional_t<Exponents, uint32_t, F32x4> Scales;  // of the weight, for four blocks
    const Scales* scales_of;
    // Every read is of memory that is there: past the weight's last tiles those again, past x's row
    // tiles what comes behind them (kPastRows), past the last block of x the last.  (What is the same for all lanes,
    // an offset in a scalar register, comes off a resource's size before the comparison, below zero
    // too: only the lanes' own offsets are guarded by it.)  None of that is stored.
    auto take = [&](int64_t number) {
        const int64_t band = number / (8 * out_groups), in_band = number - band * 8 * out_groups;
        const int64_t high = min((int64_t)8, row_groups - 8 * band);
        const int64_t out_group = in_band / high, row_group = 8 * band + in_band % high;
        tile0 = 16 * out_group + 4 * wave;
        row_tile0 = NT * row_group;
        auto resource = [](const void* base, int64_t bytes) { return handoff_resource(base, (uint32_t)bytes); };
        const int64_t own = min(tile0, out_tiles - 4);
        weights = resource(p.packed + own * blocks * kTileBytes, 4 * blocks * kTileBytes);
        x_all = resource(p.x_codes + row_tile0 * kTileBytes, (blocks * row_tiles - row_tile0) * kTileBytes + kPastRows);
        x_scales = resource(p.x_scales + row_tile0 * 16, (fours * row_tiles - row_tile0) * 64 + kPastRows);
        scales_of = reinterpret_cast<const Scales*>(p.packed_scales) + own / 8 * fours;
    };

    F32x4 total[4][NT];
    I32x8 a[2][4];
    U32x4 piece[kPieces];
    uint32_t word;  // of x's scales, on its way to LDS
    Scales w_scales;  // FP32: their factors
    uint32_t w_powers = 0;  // FP32: their powers of two, a byte each
    auto load_x = [&](int b) {
#pragma unroll
        for (int c = 0; c < kPieces; ++c)
            piece[c] = __builtin_amdgcn_raw_buffer_load_b128(x_all, 16 * tid, 4096 * c + b * x_stride, 0);
    };
    auto store_x = [&](int buffer) {
#pragma unroll
        for (int c = 0; c < kPieces; ++c) *reinterpret_cast<U32x4*>(&lds[buffer][16 * (256 * c + tid)]) = piece[c];
    };
    auto load_a = [&](I32x8 (&to)[4], int b) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // (The lane's offset holds the block, so that past the last block it is past the resource and reads 0.)
            const uint32_t at = 16 * lane + 4 * b * kTileBytes + (j & 1) * kTileBytes, pair = (j >> 1) * 2 * kTileBytes;
            const U32x4 low = __builtin_amdgcn_raw_buffer_load_b128(weights, at, pair, 0);
            const U32x4 high = __builtin_amdgcn_raw_buffer_load_b128(weights, at + 1024, pair, 0);
            to[j] = I32x8{(int)low[0], (int)low[1], (int)low[2], (int)low[3], (int)high[0], (int)high[1], (int)high[2], (int)high[3]};
        }
    };
    auto load_word = [&](int four) {
        word = __builtin_amdgcn_raw_buffer_load_b32(x_scales, 4 * tid, four * words_stride, 0);
    };
    auto store_word = [&](int four) {
        if (tid < 16 * NT) x_words[four & 1][tid] = word;
    };
    auto load_scales = [&](int four) {
        const Scales v = scales_of[four];
        if constexpr (Exponents) {
            w_scales = __builtin_amdgcn_readfirstlane(v);
        } else {
            uint32_t powers = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t power = scale_power(v[e]);
                w_scales[e] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(scale_factor(v[e], power))));
                powers |= power << (8 * e);
            }
            w_powers = powers;
        }
    };
    // Block 4 four + S.
    auto step = [&](auto place, int four) {
        constexpr int S = decltype(place)::value;
        const int b = 4 * four + S;
        store_x((S + 2) & 3);
        load_x(min(b + 3, blocks - 1));
        load_a(a[(S + 1) & 1], b + 1);
        if constexpr (S == 0) load_word(min(four + 1, fours - 1));
        if constexpr (S == 2) store_word(four + 1);
        __builtin_amdgcn_sched_barrier(0);
        const uint8_t* from = lds[S];
        const uint32_t* from_words = &x_words[four & 1][i];
        I32x8 x[2];
        uint32_t x_scale[2];
        x[0] = operand(from, lane);
        x_scale[0] = from_words[0];
        // FP32 scales: a row tile's sums are added while the next one's products run, if the registers last (of 128 rows
        // 38 would spill: right behind each product then).
        constexpr bool kLater = !Exponents && NT < 8;
        F32x4 sum[4];
        auto add = [&](int j, int t) {
            if constexpr (!Exponents)
#pragma unroll
                for (int r = 0; r < 4; ++r) total[j][t][r] = fmaf(w_scales[S], sum[j][r], total[j][t][r]);
        };
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (t + 1 < NT) {
                x[(t + 1) & 1] = operand(from + (t + 1) * kTileBytes, lane);
                x_scale[(t + 1) & 1] = from_words[16 * (t + 1)];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (Exponents) {
                    total[j][t] = mfma<S, S>(a[S & 1][j], x[t & 1], total[j][t], w_scales, x_scale[t & 1]);
                } else {
                    if (kLater && t > 0) add(j, t - 1);
                    sum[j] = mfma<S, S>(a[S & 1][j], x[t & 1], F32x4{0.f, 0.f, 0.f, 0.f}, w_powers, x_scale[t & 1]);
                    if (!kLater) add(j, t);
                }
            }
        }
        if constexpr (kLater)
#pragma unroll
            for (int j = 0; j < 4; ++j) add(j, NT - 1);
        // The operands of a row tile are read while the products of the one before run.
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            if (t < NT - 1) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
            if constexpr (kLater) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (t > 0) __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                }
            } else {
                __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
            }
        }
        if constexpr (S & 1) lds_barrier();
    };

    int64_t number = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (number >= stop) return;
    auto begin = [&] {
        take(number);
        load_x(0);
        load_a(a[0], 0);
        load_word(0);
    };
    begin();
    while (true) {
        load_scales(0);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int t = 0; t < NT; ++t) total[j][t] = F32x4{0.f, 0.f, 0.f, 0.f};
        store_x(0);
        store_word(0);
        load_x(min(1, blocks - 1));
        store_x(1);
        load_x(min(2, blocks - 1));
        lds_barrier();
        for (int four = 0; four < fours; ++four) {
            step(std::integral_constant<int, 0>{}, four);
            if (4 * four + 1 < blocks) step(std::integral_constant<int, 1>{}, four);
            if (4 * four + 2 < blocks) step(std::integral_constant<int, 2>{}, four);
            if (4 * four + 3 < blocks) step(std::integral_constant<int, 3>{}, four);
            load_scales(min(four + 1, fours - 1));
        }
        // The next tile's first block, then this one's results.
        const int64_t out_at = 16 * tile0 + 8 * g, row_at = 16 * row_tile0 + i;
        number += step_of_tiles;
        const bool more = number < stop;
        if (more) begin();
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int64_t m = row_at + 16 * t;
            if (m >= p.rows) continue;
            uint16_t* const to = p.y + m * p.y_stride + out_at;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const F32x4 u = total[2 * h][t], v = total[2 * h + 1][t];
                if (out_at + 32 * h + 8 <= p.out_features) {
                    *reinterpret_cast<U32x4At2*>(to + 32 * h) =
                        U32x4{bf16x2_rn(u[0], u[1]), bf16x2_rn(u[2], u[3]), bf16x2_rn(v[0], v[1]), bf16x2_rn(v[2], v[3])};
                    continue;
                }
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    if (out_at + 32 * h + r < p.out_features) to[32 * h + r] = (uint16_t)bf16_rn(r < 4 ? u[r] : v[r - 4]);
            }
        }
        if (!more) return;
        // (A step of the last pair may still be reading its buffers.)
        lds_barrier();
    }
}

// One workgroup per compute unit at most: x is read and rounded by each. (32 rows, 2048 -> 11264: 8.9 us, with
// two 12.3; -> 50257 24.7 and 25.1, 16 rows 21.2 and 21.1.)
template <bool Exponents, int T, int W, int B>
void launch_few_of(const LinearFp8Params& p, hipStream_t stream) {
    const unsigned grid = (unsigned)std::min<int64_t>(out_tiles_of(p.out_features), p.compute_units);
    hipLaunchKernelGGL((linear_fp8_few_kernel<T, W, B, Exponents>), dim3(grid), dim3(64 * W), 0, stream, p);
}
template <bool Exponents>
void launch_few(const LinearFp8Params& p, hipStream_t stream) {
    const int64_t blocks = blocks_of(p.in_features);
    if (p.rows > 32)
        return blocks <= 8 ? launch_few_of<Exponents, 3, 8, 1>(p, stream) : launch_few_of<Exponents, 3, 8, 2>(p, stream);
    if (p.rows > 16) {
        if (blocks <= 8) return launch_few_of<Exponents, 2, 8, 1>(p, stream);
        return blocks <= 16 ? launch_few_of<Exponents, 2, 8, 2>(p, stream) : launch_few_of<Exponents, 2, 16, 2>(p, stream);
    }
    if (blocks <= 8)
        launch_few_of<Exponents, 1, 8, 1>(p, stream);
    else if (blocks <= 16)
        launch_few_of<Exponents, 1, 8, 2>(p, stream);
    else if (blocks <= 32)
        launch_few_of<Exponents, 1, 16, 2>(p, stream);
    else if (blocks <= 48)
        launch_few_of<Exponents, 1, 16, 3>(p, stream);
    else
        launch_few_of<Exponents, 1, 16, 4>(p, stream);
}

template <bool Exponents, int J, int T>
void launch_split(const LinearFp8Params& p, hipStream_t stream) {
    const int64_t groups = out_tiles_of(p.out_features) / J * ((tiles_of(p.rows) + T - 1) / T);
    hipLaunchKernelGGL((linear_fp8_split_kernel<J, T, Exponents>), dim3((unsigned)groups), dim3(512), 0, stream, p);
}

// Two workgroups per compute unit, in whole rounds of the XCDs.
template <bool Exponents, int NT>
void launch_wide(const LinearFp8Params& p, hipStream_t stream) {
    const int64_t tiles = ((p.out_features + 255) / 256) * ((p.rows + 16 * NT - 1) / (16 * NT));
    const unsigned grid = (unsigned)std::min<int64_t>((tiles + 7) / 8 * 8, std::max(p.compute_units / 8, 1) * 16);
    hipLaunchKernelGGL((linear_fp8_wide_kernel<Exponents, NT>), dim3(grid), dim3(256), 0, stream, p);
}

// The kernel for rows in operand order: by what its rounds of workgroups take, two
// per compute unit or one in the last, a block of inputs at a time. Measured in us per
// block with one workgroup on a compute unit and with two, and per round (the join,
// the first loads; two of 64 x 64 take 256 KB of LDS and follow one another); of 38 shapes
// from 32 to 8192 rows the choice takes the fastest of the six, or up to 10% longer. Fewer rows over inputs too
// long for the kernel above are not among these: up to 16 multiply a tile of x twice (1 row, 16384 -> 2048
// 15.8 us, 16 rows 16.1, 31 rows, 8192 -> 2048 11.7). (1018 rows, 2048 -> 11264: tiles of 256 x 96 31.5 us, x 64
// 33.2, x 128 39.1, 64 x 64 74. 40 rows, 5632 -> 2048: 32 x 32 6.1, 64 x 64 10.3. 512 rows,
// 5632 -> 2048: 64 x 64 18.6, 256 x 64 30.9.)
struct Tiling {
    int outs, rows;
    float one, two, round;
};
template <bool Exponents>
int fastest_tiling(const LinearFp8Params& p) {
    constexpr Tiling kTilings[6] = {
        {32, 32, 0.10f, 0.30f, 0.3f},
        {32, 64, 0.17f, 0.36f, 0.6f},
        {64, 64, 0.27f, 0.54f, 1.2f},
        {256, 64, Exponents ? 0.55f : 0.63f, Exponents ? 1.05f : 1.13f, 0.3f},
        {256, 96, Exponents ? 0.70f : 0.85f, Exponents ? 1.45f : 1.67f, 0.3f},
        {256, 128, Exponents ? 0.85f : 1.33f, Exponents ? 1.75f : 2.15f, 0.3f},
    };
    const float blocks = (float)blocks_of(p.in_features);
    int best = 0;
    float least = 0.f;
    for (int c = 0; c < 6; ++c) {
        const Tiling& t = kTilings[c];
        const int64_t groups = ((p.out_features + t.outs - 1) / t.outs) * ((p.rows + t.rows - 1) / t.rows);
        const int64_t pairs = groups / (2 * p.compute_units), rest = groups % (2 * p.compute_units);
        const float pair = t.two * blocks + 2 * t.round;
        const float time = (float)pairs * pair + (rest > p.compute_units ? pair : rest > 0 ? t.one * blocks + t.round : 0.f);
        if (c == 0 || time < least) best = c, least = time;
    }
    return best;
}

template <bool Exponents>
void launch_product(const LinearFp8Params& p, hipStream_t stream) {
    switch (fastest_tiling<Exponents>(p)) {
        case 0: return launch_split<Exponents, 2, 2>(p, stream);
        case 1: return launch_split<Exponents, 2, 4>(p, stream);
        case 2: return launch_split<Exponents, 4, 4>(p, stream);
        case 3: return launch_wide<Exponents, 4>(p, stream);
        case 4: return launch_wide<Exponents, 6>(p, stream);
        default: return launch_wide<Exponents, 8>(p, stream);
    }
}

// Rows of one launch: the wide kernels address the codes of x in 31 bits.
int64_t rows_at_once(int64_t in_features) { return (((int64_t)1 << 31) - 1) / (blocks_of(in_features) * kBlock) / 128 * 128; }

}  // namespace

static size_t fp8_row_bytes(int64_t rows, int64_t in_features) { return (size_t)tiles_of(rows) * blocks_of(in_features) * kTileBytes; }

size_t fp8_code_bytes(int64_t out_features, int64_t in_features) {
    return (size_t)out_tiles_of(out_features) * blocks_of(in_features) * kTileBytes;
}

size_t fp8_weight_bytes(int64_t out_features, int64_t in_features, bool exponents) {
    return fp8_code_bytes(out_features, in_features) +
           (size_t)((out_features + kBlock - 1) / kBlock) * fours_of(in_features) * (exponents ? 4 : 16);
}

// Whether every workgroup rounds x for itself, or a launch before the product does:
// by x's blocks. (2048 -> 6144: 1 row 4.4 us against 6.9, 16 rows 5.4 against 7.1, 24 rows 7.1
// against 7.5, 40 rows 9.8 against 8.5; 2048 -> 2048: 32 rows 6.9 both; 5632 -> 2048: 1 row 5.9 against
// 8.8, 11 rows 7.9 against 9.0, 16 rows 9.2 against 9.1; 2048 -> 50257: 32 rows 24.5 against 26.1. At
// the most blocks the outputs decide too: 8192 inputs, 8 rows, 2048 outputs 9.6 against 10.5, 8192 outputs
// 17.2 against 15.6; the workspace would then depend on them.)
constexpr int64_t kFewMaxRows = 48, kFewMaxBlocks = 64, kFewMost = 512;
static bool few_rows(int64_t rows, int64_t in_features) {
    const int64_t blocks = blocks_of(in_features);
    return rows <= kFewMaxRows && blocks <= kFewMaxBlocks && rows * blocks <= kFewMost;
}

size_t linear_fp8_workspace(int64_t rows, int64_t in_features) {
    if (few_rows(rows, in_features)) return 0;
    rows = std::min(rows, rows_at_once(in_features));
    return fp8_row_bytes(rows, in_features) + (size_t)tiles_of(rows) * fours_of(in_features) * 64 + kPastRows;
}

hipError_t launch_pack_fp8(const Fp8PackParams& p, hipStream_t stream) {
    if (p.weight != nullptr) {
        const int64_t high = (p.out_features + kBlock - 1) / kBlock;
        hipLaunchKernelGGL(quantize_weight_fp8_kernel, dim3((unsigned)(high * blocks_of(p.in_features))), dim3(256), 0, stream, p);
    } else {
        // (128 pieces a tile: more threads than the scales, four of which a tile may pad.)
        const int64_t pieces = out_tiles_of(p.out_features) * blocks_of(p.in_features) * (kTileBytes / 16);
        hipLaunchKernelGGL(pack_fp8_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, p);
    }
    return hipGetLastError();
}

hipError_t launch_unpack_fp8(const Fp8PackParams& p, uint16_t* weight, hipStream_t stream) {
    const int64_t pieces = out_tiles_of(p.out_features) * blocks_of(p.in_features) * (kTileBytes / 16);
    hipLaunchKernelGGL(unpack_fp8_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, p, weight);
    return hipGetLastError();
}

hipError_t launch_linear_fp8(const LinearFp8Params& given, hipStream_t stream) {
    LinearFp8Params p = given;
    if (few_rows(p.rows, p.in_features)) {
        // (Whole pieces of eight inputs, within 2^31 bytes.)
        p.wide = p.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 && p.in_features % 8 == 0 &&
                 p.rows * p.x_stride < ((int64_t)1 << 30);
        p.exponents ? launch_few<true>(p, stream) : launch_few<false>(p, stream);
        return hipGetLastError();
    }
    const int64_t most = rows_at_once(p.in_features);
    for (int64_t first = 0; first < given.rows; first += most) {
        p.rows = std::min(given.rows - first, most);
        p.x = given.x + first * p.x_stride;
        p.y = given.y + first * p.y_stride;
        p.x_scales = reinterpret_cast<uint32_t*>(p.x_codes + fp8_row_bytes(p.rows, p.in_features));
        const dim3 grid((unsigned)(fours_of(p.in_features) * tiles_of(p.rows)));
        if (p.in_features % 8 == 0)
            hipLaunchKernelGGL(quantize_rows_fp8_kernel<true>, grid, dim3(256), 0, stream, p);
        else
            hipLaunchKernelGGL(quantize_rows_fp8_kernel<false>, grid, dim3(256), 0, stream, p);
        p.exponents ? launch_product<true>(p, stream) : launch_product<false>(p, stream);
    }
    return hipGetLastError();
}

}  // namespace rq
