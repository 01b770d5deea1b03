// Projections with 4-bit weights: y[m, n] = bf16(sum_g s[n, g] sum_{k in g} c[n, k] x[m, k]),
// c in -8..7, one BF16 scale per output row and group of 32, 64 or 128 inputs.
//
// Packed layout, made once from the codes: tiles of 16 output rows, in a tile
// blocks of 128 inputs of 1 KB each.  Lane l of a wave reads 16 bytes at
// 16 l: word i holds the codes of row l % 16 at inputs 32 i + 8 (l / 16) + e,
// e = 0..7 (code_shift), the A operand of v_mfma_f32_16x16x32 for 16 output
// rows.  Rows and inputs past the weight hold code 0.  The scales follow (scale_place),
// in the order in which the lanes of the product's result need them.
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

// Place of the scale of output row 16 tile + row and input group `group`:
// [tile][block of 128 inputs][row / 4][group of the block][row % 4].
__device__ __forceinline__ int64_t scale_place(int64_t tile, int64_t blocks, int64_t group, int group_size, int row) {
    const int per = 128 / group_size;
    return (((tile * blocks + group / per) * 4 + (row >> 2)) * per + group % per) * 4 + (row & 3);
}

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
    uint32_t scale_bits = 0;
    if (inside) {
        const int64_t group = k / p.group, groups = p.in_features / p.group;
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
    }
    if (k % p.group == 0)
        p.packed_scales[scale_place(tile, blocks, k / p.group, p.group, lane & 15)] = (uint16_t)scale_bits;
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
    const float scale = bf16_f32(p.packed_scales[scale_place(tile, blocks, k / p.group, p.group, lane & 15)]);
    for (int e = 0; e < 8; ++e)
        weight[n * p.in_features + k + e] = (uint16_t)bf16_rn((float)code_at(p.packed[w], e) * scale);
}

typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef float F32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ F32x4 mfma(U32x4 a, U32x4 b, F32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0, 0, 0);
}

// The eight codes of a word as BF16 numbers 1 + (c + 8) / 16, in three shifts
// and four v_and_or: a code takes the upper four mantissa bits of a 1.
__device__ __forceinline__ U32x4 codes_bf16(uint32_t word) {
    constexpr uint32_t kMantissa = 0x00780078u, kOne = 0x3f803f80u;
    return U32x4{(word & kMantissa) | kOne, ((word >> 4) & kMantissa) | kOne, ((word >> 8) & kMantissa) | kOne,
                 (__builtin_amdgcn_alignbit(word, word, 12) & kMantissa) | kOne};
}

// y of the outputs 16 tile0.. of NB tiles in plain steps, for results that are
// not finite: the products of shifted codes overflow earlier than the sum
// itself, and turn an infinity in x into NaN.
__device__ void linear_int4_plain(const LinearInt4Params& p, int64_t tile0, int tiles, int threads) {
    const int64_t blocks = int4_blocks(p.in_features);
    for (int64_t o = threadIdx.x; o < (int64_t)tiles * 16 * p.rows; o += threads) {
        const int64_t tile = tile0 + o / 16 % tiles, n = 16 * tile + o % 16, m = o / (16 * tiles);
        if (n >= p.out_features) continue;
        float sum = 0.f;
        for (int64_t k = 0; k < p.in_features; k += 8) {
            const uint32_t word = p.packed[((tile * blocks + k / 128) * 64 + (n & 15) + 16 * (k / 8 % 4)) * 4 + k / 32 % 4];
            const float scale = bf16_f32(p.packed_scales[scale_place(tile, blocks, k / p.group, p.group, (int)(n & 15))]);
            for (int e = 0; e < 8; ++e) sum += (float)code_at(word, e) * (bf16_f32(p.x[m * p.x_stride + k + e]) * scale);
        }
        p.y[m * p.y_stride + n] = (uint16_t)bf16_rn(sum);
    }
}

// y of every output in plain steps, for strides past what the buffer loads of x address.
__global__ __launch_bounds__(256) void linear_int4_plain_kernel(const LinearInt4Params p) {
    linear_int4_plain(p, blockIdx.x, 1, 256);
}

// One workgroup per NB tiles of 16 outputs, for all rows (T tiles of 16).  Its
// W waves share the inputs out in blocks of 128.  With u = c + 8 and
// v = 1 + u / 16 (codes_bf16), sum c x = 16 (sum v x - 1.5 sum x): the second
// sum, from a constant operand, is the accumulator that the first starts with,
// once per group for all tiles.  The next block's loads are in flight during a
// block's products; x is read by buffer loads, which give 0 to lanes past its
// rows without a branch per load.
template <int Group, int T, int NB, int W>
__global__ __launch_bounds__(64 * W) void linear_int4_kernel(const LinearInt4Params p) {
    constexpr int kPer = 128 / Group, kGroupSteps = Group / 32;
    __shared__ F32x4 partial[W][NB][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int in_features = (int)p.in_features, blocks = (int)int4_blocks(p.in_features);
    const int64_t tiles = int4_tiles(p.out_features);
    const int64_t tile0 = (int64_t)blockIdx.x * NB;
    const int begin = blocks * wave / W, end = blocks * (wave + 1) / W;
    F32x4 total[NB][T];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int t = 0; t < T; ++t) total[j][t] = F32x4{0.f, 0.f, 0.f, 0.f};
    // (The host takes other strides to linear_int4_plain_kernel.)
    const uint32_t x_bytes = (uint32_t)((p.rows - 1) * p.x_stride + p.in_features) * 2;
    const __amdgpu_buffer_rsrc_t x_rows = handoff_resource(p.x, x_bytes);
    constexpr uint32_t kOutside = 0xfffffff0u;
    uint32_t x_place[T];
#pragma unroll
    for (int t = 0; t < T; ++t) x_place[t] = 16 * t + i < p.rows ? (uint32_t)((16 * t + i) * p.x_stride + 8 * g) * 2 : kOutside;
    struct Codes {
        U32x4 words[NB];
        uint32_t scales[NB][2 * kPer];
    };
    struct Inputs {
        U32x4 x[T][4];
    };
    auto load_codes = [&](Codes& b, int block) {
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int64_t place = min(tile0 + j, tiles - 1) * blocks + block;
            b.words[j] = __builtin_nontemporal_load(reinterpret_cast<const U32x4*>(p.packed) + place * 64 + lane);
            const uint32_t* scales = reinterpret_cast<const uint32_t*>(p.packed_scales) + place * (8 * kPer) + g * (2 * kPer);
            if constexpr (kPer == 1) {
                const uint2 v = *reinterpret_cast<const uint2*>(scales);
                b.scales[j][0] = v.x, b.scales[j][1] = v.y;
            } else {
#pragma unroll
                for (int h = 0; h < kPer / 2; ++h) {
                    const U32x4 v = *reinterpret_cast<const U32x4*>(scales + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) b.scales[j][4 * h + e] = v[e];
                }
            }
        }
    };
    auto load_inputs = [&](Inputs& b, int block) {
        const bool whole = 128 * block + 128 <= in_features;
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                uint32_t place = x_place[t] + 64 * s;
                if (16 * t + i >= p.rows || (!whole && 128 * block + 32 * s + 8 * g >= in_features)) place = kOutside;
                b.x[t][s] = __builtin_amdgcn_raw_buffer_load_b128(x_rows, place, 256 * block, 0);
            }
    };
    auto compute = [&](const Codes& b, const Inputs& in) {
        const U32x4 shift = {0xbfc0bfc0u, 0xbfc0bfc0u, 0xbfc0bfc0u, 0xbfc0bfc0u};  // -1.5
#pragma unroll
        for (int h = 0; h < kPer; ++h) {
            F32x4 start[T];
#pragma unroll
            for (int t = 0; t < T; ++t) {
                start[t] = F32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < kGroupSteps; ++s) start[t] = mfma(shift, in.x[t][h * kGroupSteps + s], start[t]);
            }
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                F32x4 sum[T];
#pragma unroll
                for (int t = 0; t < T; ++t) sum[t] = start[t];
#pragma unroll
                for (int s = 0; s < kGroupSteps; ++s) {
                    const U32x4 a = codes_bf16(b.words[j][h * kGroupSteps + s]);
#pragma unroll
                    for (int t = 0; t < T; ++t) sum[t] = mfma(a, in.x[t][h * kGroupSteps + s], sum[t]);
                }
                const uint32_t low = b.scales[j][2 * h], high = b.scales[j][2 * h + 1];
                const float scale[4] = {__uint_as_float(low << 16), __uint_as_float(low & 0xffff0000u),
                                        __uint_as_float(high << 16), __uint_as_float(high & 0xffff0000u)};
#pragma unroll
                for (int t = 0; t < T; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) total[j][t][r] = fmaf(scale[r], sum[t][r], total[j][t][r]);
            }
        }
    };
    if (begin < end) {
        Codes codes;
        Inputs inputs;
        load_codes(codes, begin);
        load_inputs(inputs, begin);
        // (Rolled: a wave runs two to six rounds, and code that runs once is fetched as it runs.)
#pragma unroll 1
        for (int b = begin; b < end; ++b) {
            Codes next_codes = codes;
            Inputs next_inputs = inputs;
            if (b + 1 < end) {
                load_codes(next_codes, b + 1);
                load_inputs(next_inputs, b + 1);
            }
            compute(codes, inputs);
            codes = next_codes;
            inputs = next_inputs;
        }
    }
    bool finite = true;
#pragma unroll
    for (int t = 0; t < T; ++t) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int j = 0; j < NB; ++j) partial[wave][j][lane] = total[j][t];
        __syncthreads();
        const int j = wave;
        if (j < NB) {
            F32x4 sum = partial[0][j][lane];
#pragma unroll
            for (int w = 1; w < W; ++w) sum += partial[w][j][lane];
            const int64_t n = 16 * (tile0 + j) + 4 * g, m = 16 * t + i;
            if (m < p.rows) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (n + r >= p.out_features) break;
                    finite = finite && fabsf(sum[r]) < __builtin_inff();
                    p.y[m * p.y_stride + n + r] = (uint16_t)bf16_rn(16.0f * sum[r]);
                }
            }
        }
    }
    if (__syncthreads_or(!finite)) linear_int4_plain(p, tile0, (int)min((int64_t)NB, tiles - tile0), 64 * W);
}

template <int Group, int T>
void launch_tiles(const LinearInt4Params& p, hipStream_t stream) {
    const int64_t tiles = int4_tiles(p.out_features);
    if (tiles >= 1024)
        hipLaunchKernelGGL((linear_int4_kernel<Group, T, 4, 4>), dim3((unsigned)((tiles + 3) / 4)), dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((linear_int4_kernel<Group, T, 1, 8>), dim3((unsigned)tiles), dim3(512), 0, stream, p);
}

template <int Group>
void launch_rows(const LinearInt4Params& p, hipStream_t stream) {
    switch ((p.rows + 15) / 16) {
        case 1: return launch_tiles<Group, 1>(p, stream);
        case 2: return launch_tiles<Group, 2>(p, stream);
        case 3: return launch_tiles<Group, 3>(p, stream);
        default: return launch_tiles<Group, 4>(p, stream);
    }
}

}  // namespace

size_t int4_code_bytes(int64_t out_features, int64_t in_features) {
    return (size_t)int4_tiles(out_features) * int4_blocks(in_features) * 1024;
}

size_t int4_weight_bytes(int64_t out_features, int64_t in_features, int group) {
    return int4_code_bytes(out_features, in_features) + (size_t)int4_tiles(out_features) * int4_blocks(in_features) * (128 / group) * 32;
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
    if (p.x_stride >= (1 << 24))  // 64 rows would pass the 2 GiB that the buffer loads of x address
        hipLaunchKernelGGL(linear_int4_plain_kernel, dim3((unsigned)int4_tiles(p.out_features)), dim3(256), 0, stream, p);
    else if (p.group == 32)
        launch_rows<32>(p, stream);
    else if (p.group == 64)
        launch_rows<64>(p, stream);
    else
        launch_rows<128>(p, stream);
    return hipGetLastError();
}

}  // namespace rq
