// Projections in 8-bit floating point: with E4M3 codes c and block scales s,
//   y[m, n] = bf16(sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} cx[m, k] cw[n, k]),
// blocks of 128 inputs.  sx[m, b] is the least power of two >= 2^-126 with
// |x| <= 448 sx for the block's finite values, cx = x / sx to nearest, ties to
// even; sw is given for 128 outputs x 128 inputs, as an exponent (E8M0) or in FP32.
//
// Both operands lie in tiles of 16 rows x 128 inputs, 2 KB each, in the order in
// which v_mfma_scale_f32_16x16x128 takes them: lane l = (i = l % 16, g = l / 16)
// holds row i, inputs 32 g + 16 h + 0..15 in the 16 bytes at 1024 h + 16 l, h = 0,
// 1.  (An instruction sums over all 128 inputs, so their order matters only in
// that both operands have the same.)  Rows and inputs past the matrix hold 0.
// The instruction multiplies by powers of two as it goes: sx always, sw if it
// is an exponent; an FP32 sw multiplies each block's FP32 sum instead.
//
// What the 8-bit instructions cost in exactness: beside FP32 sums they line 16
// products up with the largest and cut what lies below 2^-13 of its power of two.
// Against sums in 64 bits results are off by 1.4e-5 (normal values) to 5.6e-5 (codes of
// all sizes) in the 2-norm, at 128 as at 2048 inputs, a hundredth of what the
// rounding to BF16 is off by (1.7e-3). v_mfma_f32_16x16x32_fp8_fp8 cuts alike;
// codes converted to BF16 operands would not (3e-7), at half the rate and with a
// conversion per two codes.
#include <algorithm>

#include "rq_device.h"
#include "rq_fp8.h"
#include "rq_reduced.h"

namespace rq {

namespace {

typedef float F32x4 __attribute__((ext_vector_type(4)));
typedef int I32x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = 128, kTileBytes = 16 * kBlock;

__host__ __device__ __forceinline__ int64_t tiles_of(int64_t rows) { return (rows + 15) / 16; }
__host__ __device__ __forceinline__ int64_t blocks_of(int64_t in_features) { return (in_features + kBlock - 1) / kBlock; }
// Scales lie in fours, one word per row (or block row) and four blocks.
__host__ __device__ __forceinline__ int64_t fours_of(int64_t in_features) { return (blocks_of(in_features) + 3) / 4; }

// The exponent byte (E8M0, 2^(byte - 127)) of a block's scale.
__device__ __forceinline__ int scale_exponent(float largest) { return (int)(__float_as_uint(needed_scale(largest)) >> 23); }
// 2^(127 - byte): what a value is multiplied by before its rounding, exactly (byte <= 247).
__device__ __forceinline__ float inverse_scale(int exponent) { return __uint_as_float((uint32_t)(254 - exponent) << 23); }

__device__ __forceinline__ float finite_size(float x) { return fabsf(x) < __builtin_inff() ? fabsf(x) : 0.f; }

// ------------------------------------------------------------------ weights

// One thread per 16 bytes of the packed codes.
__global__ __launch_bounds__(256) void pack_fp8_kernel(const Fp8PackParams p) {
    const int64_t blocks = blocks_of(p.in_features), pieces = tiles_of(p.out_features) * blocks * (kTileBytes / 16);
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
    const int64_t block = (w >> 7) % blocks, n = 16 * ((w >> 7) / blocks) + (lane & 15);
    const int64_t k = kBlock * block + 32 * (lane >> 4) + 16 * half;
    U32x4 piece = {0u, 0u, 0u, 0u};
    if (n < p.out_features)
        for (int e = 0; e < 16; ++e)
            if (k + e < p.in_features) piece[e >> 2] |= (uint32_t)p.codes[n * p.in_features + k + e] << (8 * (e & 3));
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
    const int64_t tiles = tiles_of(p.out_features);
    for (int w = threadIdx.x; w < 8 * (kTileBytes / 16); w += 256) {
        const int lane = w & 63, half = (w >> 6) & 1;
        const int64_t tile = 8 * high + (w >> 7), n = 16 * tile + (lane & 15), k = kBlock * block + 32 * (lane >> 4) + 16 * half;
        if (tile >= tiles) continue;
        float x[16];
        for (int e = 0; e < 16; ++e)
            x[e] = n < p.out_features && k + e < p.in_features ? bf16_f32(p.weight[n * p.in_features + k + e]) * inverse : 0.f;
        U32x4 piece;
        for (int e = 0; e < 4; ++e) piece[e] = fp8x4_rn(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
        reinterpret_cast<U32x4*>(p.packed)[((tile * blocks + block) * 2 + half) * 64 + lane] = piece;
    }
}

// The BF16 weight [out, in] of a packed one: bf16(code x scale).  One thread per 16 bytes.
__global__ __launch_bounds__(256) void unpack_fp8_kernel(const Fp8PackParams p, uint16_t* weight) {
    const int64_t blocks = blocks_of(p.in_features), pieces = tiles_of(p.out_features) * blocks * (kTileBytes / 16);
    const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (w >= pieces) return;
    const int lane = (int)w & 63, half = (int)(w >> 6) & 1;
    const int64_t block = (w >> 7) % blocks, n = 16 * ((w >> 7) / blocks) + (lane & 15);
    const int64_t k = kBlock * block + 32 * (lane >> 4) + 16 * half;
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
    for (int e = 0; e < 16 && k + e < p.in_features; ++e)
        weight[n * p.in_features + k + e] = (uint16_t)bf16_rn(e4m3_f32((piece[e >> 2] >> (8 * (e & 3))) & 0xffu) * scale);
}

// ------------------------------------------------------------------ rows

// One workgroup per tile of 16 rows and four blocks of 128 inputs; 16 lanes per row of a block.
template <bool Wide>
__global__ __launch_bounds__(256) void quantize_rows_fp8_kernel(const LinearFp8Params p) {
    const int tid = threadIdx.x, j = tid & 15, i = tid >> 4;
    const int64_t blocks = blocks_of(p.in_features), fours = fours_of(p.in_features);
    const int64_t four = blockIdx.x % fours, tile = blockIdx.x / fours, m = 16 * tile + i;
    const uint16_t* row = p.x + m * p.x_stride;
    uint32_t word = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int64_t block = 4 * four + b, k = kBlock * block + 8 * j;
        float x[8];
        if (Wide && m < p.rows && k + 8 <= p.in_features) {
            const U32x4 raw = *reinterpret_cast<const U32x4*>(row + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[2 * e] = __uint_as_float(raw[e] << 16);
                x[2 * e + 1] = __uint_as_float(raw[e] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = m < p.rows && k + e < p.in_features ? bf16_f32(row[k + e]) : 0.f;
        }
        float largest = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) largest = fmaxf(largest, finite_size(x[e]));
#pragma unroll
        for (int d = 8; d; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
        const int exponent = scale_exponent(largest);
        const float inverse = inverse_scale(exponent);
        word |= (uint32_t)exponent << (8 * b);
        if (block < blocks) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= inverse;
            const uint2 codes = make_uint2(fp8x4_rn(x[0], x[1], x[2], x[3]), fp8x4_rn(x[4], x[5], x[6], x[7]));
            uint8_t* to = p.x_codes + (tile * blocks + block) * kTileBytes;
            *reinterpret_cast<uint2*>(to + 1024 * ((j >> 1) & 1) + 16 * (i + 16 * (j >> 2)) + 8 * (j & 1)) = codes;
        }
    }
    if (j == 0) p.x_scales[(tile * fours + four) * 16 + i] = word;
}

// ------------------------------------------------------------------ product

__device__ __forceinline__ I32x8 operand(const uint8_t* tile, int lane) {
    const U32x4 a = *reinterpret_cast<const U32x4*>(tile + 16 * lane), b = *reinterpret_cast<const U32x4*>(tile + 1024 + 16 * lane);
    return I32x8{(int)a[0], (int)a[1], (int)a[2], (int)a[3], (int)b[0], (int)b[1], (int)b[2], (int)b[3]};
}

// 16 outputs (a) x 16 rows (b) over 128 inputs; lane (i, g) of the result: row i, outputs 4 g + 0..3.
__device__ __forceinline__ F32x4 mfma(I32x8 a, I32x8 b, F32x4 c, uint32_t scale_a, uint32_t scale_b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, (int)scale_a, 0, (int)scale_b);
}

// One workgroup of eight waves per 16 outputs and T tiles of 16 rows; the waves share the inputs out.
template <int T, bool Exponents>
__global__ __launch_bounds__(512) void linear_fp8_kernel(const LinearFp8Params p) {
    __shared__ F32x4 partial[8][T][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int blocks = (int)blocks_of(p.in_features), fours = (int)fours_of(p.in_features);
    const int64_t tile = blockIdx.x, row_tiles = tiles_of(p.rows), first = (int64_t)blockIdx.y * T;
    const int begin = blocks * wave / 8, end = blocks * (wave + 1) / 8;
    F32x4 total[T];
#pragma unroll
    for (int t = 0; t < T; ++t) total[t] = F32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t scales = tile / 8 * (4 * fours);
    for (int b = begin; b < end; ++b) {
        const I32x8 a = operand(p.packed + (tile * blocks + b) * kTileBytes, lane);
#pragma unroll
        for (int t = 0; t < T; ++t) {
            const int64_t m = min(first + t, row_tiles - 1);
            const I32x8 x = operand(p.x_codes + (m * blocks + b) * kTileBytes, lane);
            const uint32_t x_scale = p.x_scales[(m * fours + (b >> 2)) * 16 + i] >> (8 * (b & 3));
            if constexpr (Exponents) {
                total[t] = mfma(a, x, total[t], p.packed_scales[scales + b], x_scale);
            } else {
                const F32x4 sum = mfma(a, x, F32x4{0.f, 0.f, 0.f, 0.f}, 127u, x_scale);
                const float scale = reinterpret_cast<const float*>(p.packed_scales)[scales + b];
#pragma unroll
                for (int r = 0; r < 4; ++r) total[t][r] = fmaf(scale, sum[r], total[t][r]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) partial[wave][t][lane] = total[t];
    __syncthreads();
    for (int t = wave; t < T; t += 8) {
        F32x4 sum = partial[0][t][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) sum += partial[w][t][lane];
        const int64_t n = 16 * tile + 4 * g, m = 16 * (first + t) + i;
        if (m >= p.rows) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n + r < p.out_features) p.y[m * p.y_stride + n + r] = (uint16_t)bf16_rn(sum[r]);
    }
}

template <bool Exponents>
void launch_product(const LinearFp8Params& p, hipStream_t stream) {
    const int64_t row_tiles = tiles_of(p.rows);
    const unsigned tiles = (unsigned)tiles_of(p.out_features);
    if (row_tiles == 1)
        hipLaunchKernelGGL((linear_fp8_kernel<1, Exponents>), dim3(tiles), dim3(512), 0, stream, p);
    else if (row_tiles == 2)
        hipLaunchKernelGGL((linear_fp8_kernel<2, Exponents>), dim3(tiles), dim3(512), 0, stream, p);
    else
        hipLaunchKernelGGL((linear_fp8_kernel<4, Exponents>), dim3(tiles, (unsigned)((row_tiles + 3) / 4)), dim3(512), 0, stream, p);
}

}  // namespace

size_t fp8_code_bytes(int64_t rows, int64_t in_features) { return (size_t)tiles_of(rows) * blocks_of(in_features) * kTileBytes; }

size_t fp8_weight_bytes(int64_t out_features, int64_t in_features, bool exponents) {
    return fp8_code_bytes(out_features, in_features) +
           (size_t)((out_features + kBlock - 1) / kBlock) * fours_of(in_features) * (exponents ? 4 : 16);
}

size_t linear_fp8_workspace(int64_t rows, int64_t in_features) {
    return fp8_code_bytes(rows, in_features) + (size_t)tiles_of(rows) * fours_of(in_features) * 64;
}

hipError_t launch_pack_fp8(const Fp8PackParams& p, hipStream_t stream) {
    if (p.weight != nullptr) {
        const int64_t high = (p.out_features + kBlock - 1) / kBlock;
        hipLaunchKernelGGL(quantize_weight_fp8_kernel, dim3((unsigned)(high * blocks_of(p.in_features))), dim3(256), 0, stream, p);
    } else {
        // (128 pieces a tile: more threads than the scales, four of which a tile may pad.)
        const int64_t pieces = tiles_of(p.out_features) * blocks_of(p.in_features) * (kTileBytes / 16);
        hipLaunchKernelGGL(pack_fp8_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, p);
    }
    return hipGetLastError();
}

hipError_t launch_unpack_fp8(const Fp8PackParams& p, uint16_t* weight, hipStream_t stream) {
    const int64_t pieces = tiles_of(p.out_features) * blocks_of(p.in_features) * (kTileBytes / 16);
    hipLaunchKernelGGL(unpack_fp8_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, p, weight);
    return hipGetLastError();
}

hipError_t launch_linear_fp8(const LinearFp8Params& p, hipStream_t stream) {
    const dim3 grid((unsigned)(fours_of(p.in_features) * tiles_of(p.rows)));
    const bool wide = p.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0;
    if (wide)
        hipLaunchKernelGGL(quantize_rows_fp8_kernel<true>, grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL(quantize_rows_fp8_kernel<false>, grid, dim3(256), 0, stream, p);
    if (p.exponents)
        launch_product<true>(p, stream);
    else
        launch_product<false>(p, stream);
    return hipGetLastError();
}

}  // namespace rq
