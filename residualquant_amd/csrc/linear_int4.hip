// Projections with 4-bit weights: y[m, n] = bf16(sum_g s[n, g] sum_{k in g} c[n, k] x[m, k]),
// c in -8..7, one BF16 scale per output row and group of 32, 64 or 128 inputs.
//
// Packed layout, made once from the codes: tiles of 16 output rows, in a tile
// blocks of 128 inputs of 1 KB each.  Lane l of a wave reads 16 bytes at
// 16 l: word i holds the codes of row l % 16 at inputs 32 i + 8 (l / 16) + e,
// e = 0..7 (code_shift).  Rows and inputs past the weight hold code 0.  The
// scales follow: [tile][group][16 rows].
#include "rq_device.h"
#include "rq_reduced.h"

namespace rq {

namespace {

// The lowest bit of code e in its word.  The codes (plus 8, unsigned) of e =
// 0, 2, 4, 6 fill the lower and of 1, 3, 5, 7 the upper half word, and the word
// is rotated left by 3: the pair (0, 1) stands at bits 3 and 19, in the upper
// mantissa bits of two BF16 numbers.
__device__ __forceinline__ int code_shift(int e) { return (3 + 4 * (e >> 1) + 16 * (e & 1)) & 31; }

__device__ __forceinline__ uint32_t rotate_left(uint32_t x, int n) {
    n &= 31;
    return n == 0 ? x : (x << n) | (x >> (32 - n));
}

__device__ __forceinline__ int code_at(uint32_t word, int e) {
    return (int)(rotate_left(word, 32 - code_shift(e)) & 15u) - 8;
}

__host__ __device__ __forceinline__ int64_t int4_tiles(int64_t out_features) { return (out_features + 15) / 16; }
__host__ __device__ __forceinline__ int64_t int4_blocks(int64_t in_features) { return (in_features + 127) / 128; }

// One thread per word.  From codes (int8 [out, in]) and scales, or from a BF16
// weight: scale = bf16(largest |w| of the group / 7), code = round to even of
// w / scale, limited to -8..7 (0 where the scale is 0).
__global__ __launch_bounds__(256) void pack_int4_kernel(const Int4PackParams p) {
    const int64_t blocks = int4_blocks(p.in_features), words = int4_tiles(p.out_features) * blocks * 256;
    const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (w >= words) return;
    const int i = (int)(w & 3), lane = (int)(w >> 2) & 63;
    const int64_t block = (w >> 8) % blocks, tile = (w >> 8) / blocks;
    const int64_t n = 16 * tile + (lane & 15), k = 128 * block + 32 * i + 8 * (lane >> 4);
    uint32_t word = 0;
    const bool inside = n < p.out_features && k < p.in_features;
    float scale = 0.f;
    if (inside) {
        const int64_t group = k / p.group, groups = p.in_features / p.group;
        uint32_t scale_bits;
        if (p.weight != nullptr) {
            float largest = 0.f;
            for (int e = 0; e < p.group; ++e) {
                const float a = fabsf(bf16_f32(p.weight[n * p.in_features + group * p.group + e]));
                if (a > largest || a != a) largest = a;  // a NaN stays
            }
            scale_bits = bf16_rn(largest / 7.0f);
        } else {
            scale_bits = p.scales[n * groups + group];
        }
        scale = bf16_f32(scale_bits);
        if (k % p.group == 0) p.packed_scales[(tile * groups + group) * 16 + (lane & 15)] = (uint16_t)scale_bits;
    } else if (n >= p.out_features && k < p.in_features && k % p.group == 0) {
        p.packed_scales[(tile * (p.in_features / p.group) + k / p.group) * 16 + (lane & 15)] = 0;
    }
    for (int e = 0; e < 8; ++e) {
        int code = 0;
        if (inside && p.weight != nullptr) {
            const float q = rintf(bf16_f32(p.weight[n * p.in_features + k + e]) / scale);
            code = q == q ? (int)fminf(fmaxf(q, -8.f), 7.f) : 0;
        } else if (inside) {
            code = min(max((int)p.codes[n * p.in_features + k + e], -8), 7);
        }
        word |= rotate_left((uint32_t)(code + 8), code_shift(e));
    }
    p.packed[w] = word;
}

// BF16 weight [out, in] of a packed one: bf16(code * scale).  One thread per word.
__global__ __launch_bounds__(256) void unpack_int4_kernel(const Int4PackParams p, uint16_t* weight) {
    const int64_t blocks = int4_blocks(p.in_features), words = int4_tiles(p.out_features) * blocks * 256;
    const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (w >= words) return;
    const int i = (int)(w & 3), lane = (int)(w >> 2) & 63;
    const int64_t block = (w >> 8) % blocks, tile = (w >> 8) / blocks;
    const int64_t n = 16 * tile + (lane & 15), k = 128 * block + 32 * i + 8 * (lane >> 4);
    if (n >= p.out_features || k >= p.in_features) return;
    const float scale = bf16_f32(p.packed_scales[(tile * (p.in_features / p.group) + k / p.group) * 16 + (lane & 15)]);
    for (int e = 0; e < 8; ++e)
        weight[n * p.in_features + k + e] = (uint16_t)bf16_rn((float)code_at(p.packed[w], e) * scale);
}

// One wave per (tile of 16 output rows, row of x): a lane sums its 8 inputs of
// every 32, the four lanes of an output row meet at the end.
__global__ __launch_bounds__(64) void linear_int4_kernel(const LinearInt4Params p) {
    const int lane = threadIdx.x;
    const int64_t tile = blockIdx.x, row = blockIdx.y;
    const int64_t blocks = int4_blocks(p.in_features);
    const int groups = (int)(p.in_features / p.group);
    const uint16_t* x = p.x + row * p.x_stride;
    float sum = 0.f;
    for (int64_t step = 0; step < p.in_features / 32; ++step) {
        const uint32_t word = p.packed[((tile * blocks + step / 4) * 64 + lane) * 4 + (step & 3)];
        const int64_t k = 32 * step + 8 * (lane >> 4);
        const float scale = bf16_f32(p.packed_scales[(tile * groups + k / p.group) * 16 + (lane & 15)]);
        for (int e = 0; e < 8; ++e) sum += (float)code_at(word, e) * (bf16_f32(x[k + e]) * scale);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    const int64_t n = 16 * tile + (lane & 15);
    if (lane < 16 && n < p.out_features) p.y[row * p.y_stride + n] = (uint16_t)bf16_rn(sum);
}

}  // namespace

size_t int4_code_bytes(int64_t out_features, int64_t in_features) {
    return (size_t)int4_tiles(out_features) * int4_blocks(in_features) * 1024;
}

size_t int4_weight_bytes(int64_t out_features, int64_t in_features, int group) {
    return int4_code_bytes(out_features, in_features) + (size_t)int4_tiles(out_features) * (in_features / group) * 32;
}

hipError_t launch_pack_int4(const Int4PackParams& p, hipStream_t stream) {
    const int64_t words = int4_tiles(p.out_features) * int4_blocks(p.in_features) * 256;
    hipLaunchKernelGGL(pack_int4_kernel, dim3((unsigned)(words / 256)), dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_unpack_int4(const Int4PackParams& p, uint16_t* weight, hipStream_t stream) {
    const int64_t words = int4_tiles(p.out_features) * int4_blocks(p.in_features) * 256;
    hipLaunchKernelGGL(unpack_int4_kernel, dim3((unsigned)(words / 256)), dim3(256), 0, stream, p, weight);
    return hipGetLastError();
}

hipError_t launch_linear_int4(const LinearInt4Params& p, hipStream_t stream) {
    hipLaunchKernelGGL(linear_int4_kernel, dim3((unsigned)int4_tiles(p.out_features), (unsigned)p.rows), dim3(64), 0,
                       stream, p);
    return hipGetLastError();
}

}  // namespace rq
