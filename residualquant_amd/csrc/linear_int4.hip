// Projections with 4-bit weights: y[m, n] = bf16(sum_g s[n, g] sum_{k in g} c[n, k] x[m, k]),
// c in -8..7, one BF16 scale per output row and group of 32, 64 or 128 inputs.
//
// Packed layout, made once from the codes: tiles of 16 output rows, in a tile
// blocks of 128 inputs of 1 KB each.  Lane l of a wave reads 16 bytes at
// 16 l: word i holds the codes of row l % 16 at inputs 32 i + 8 (l / 16) + e,
// e = 0..7 (code_word), the A operand of v_mfma_f32_16x16x32 for 16 output
// rows.  Rows and inputs past the weight hold code 0.  The scales follow (scale_place),
// in the order in which the lanes of the product's result need them.
#include <algorithm>

#include "rq_device.h"
#include "rq_reduced.h"

namespace rq {

namespace {

__device__ __forceinline__ uint32_t rotate_right(uint32_t x, int n) { return __builtin_amdgcn_alignbit(x, x, n); }

// Code c as element e of its word: a sign s and three bits m, c = m or -m - 1.
// Elements 0..3 have m in the lowest bits and s in the top bit of byte e, 4..7
// the same after a rotation by 4 bits (code_bytes).
__device__ __forceinline__ uint32_t code_word(int c, int e) {
    const uint32_t byte = c < 0 ? 0x80u | (uint32_t)(-c - 1) : (uint32_t)c, word = byte << (8 * (e & 3));
    return e < 4 ? word : rotate_right(word, 28);
}

__device__ __forceinline__ int code_at(uint32_t word, int e) {
    const uint32_t byte = (e < 4 ? word : rotate_right(word, 4)) >> (8 * (e & 3));
    const int m = (int)(byte & 7u);
    return byte & 0x80u ? -m - 1 : m;
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
        word |= code_word(code, e);
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

// Two E4M3 bytes (of the low or high half word of x) as two BF16, exactly.
template <bool High>
__device__ __forceinline__ uint32_t bf16x2_of_fp8(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, High));
}

// Four codes as E4M3 bytes of c x 2^-9: bytes 0..15 are the multiples 0..15 of
// 2^-9 (the lowest exponents of E4M3 are linear), so the byte of |c| is |c|
// itself, m + s, below the sign.
__device__ __forceinline__ uint32_t code_bytes(uint32_t word) {
    return (word & 0x87878787u) + ((word >> 7) & 0x01010101u);
}

// The eight codes of a word as BF16 numbers c x 2^-9, each exact: 13 vector
// instructions.  (Seven make 1 + (c + 8) / 16, and c x from it less 1.5 x: then
// every input counts with 24 times its size, also under a code of 0, and one
// that is not finite takes the other codes' sums with it.)
__device__ __forceinline__ U32x4 codes_bf16(uint32_t word) {
    const uint32_t low = code_bytes(word), high = code_bytes(rotate_right(word, 4));
    return U32x4{bf16x2_of_fp8<false>(low), bf16x2_of_fp8<true>(low), bf16x2_of_fp8<false>(high), bf16x2_of_fp8<true>(high)};
}
constexpr float kCodeUnit = 512.0f;  // of the sums

// One workgroup of eight waves per 8 / WK x NB tiles of 16 outputs, for all
// rows (T tiles of 16).  x passes through LDS, in chunks of `chunk_blocks`
// blocks of 128 inputs (all of them where they fit): rows of a large power of
// two lie in one channel of the cache, so 16 rows read side by side by every
// wave took most of the time (64 rows x 16 outputs x 2048 inputs, one
// workgroup: 10.3 us, 8 of them for x).  WK waves share a tile's inputs out; a
// wave keeps the codes of kAhead blocks in flight.
typedef __attribute__((address_space(3))) void LdsVoid;

// One DMA load: lane l's 16 bytes at `offset` of the resource go to lds + 16 l (lds wave-uniform).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, uint8_t* lds, uint32_t offset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LdsVoid*)lds, 16, offset, 0, 0, 0);
}

constexpr int kLinearInt4Threads = 512;
constexpr int kRowPad = 16;  // bytes between the rows in LDS: operand reads of 16 rows meet different banks

template <int Group, int T, int NB, int WK>
__global__ __launch_bounds__(kLinearInt4Threads) void linear_int4_kernel(const LinearInt4Params p) {
    constexpr int kPer = 128 / Group, kGroupSteps = Group / 32, kAhead = NB == 1 ? 4 : 2;
    extern __shared__ __align__(16) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int part = wave % WK, rows = (int)p.rows;
    const int in_features = (int)p.in_features, blocks = (int)int4_blocks(p.in_features);
    const int64_t tiles = int4_tiles(p.out_features);
    const int64_t tile0 = ((int64_t)blockIdx.x * (8 / WK) + wave / WK) * NB;
    const int row_bytes = (p.chunk_blocks + 3) / 4 * 1024 + kRowPad;
    F32x4 total[NB][T];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int t = 0; t < T; ++t) total[j][t] = F32x4{0.f, 0.f, 0.f, 0.f};
    struct Codes {
        U32x4 words[NB];
        uint32_t scales[NB][2 * kPer];
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
    // Rows past the last read the last again; their outputs are not stored.
    const uint8_t* x_row[T];
#pragma unroll
    for (int t = 0; t < T; ++t) x_row[t] = lds + min(16 * t + i, rows - 1) * row_bytes + 16 * g;
    auto compute = [&](const Codes& b, int block) {
        U32x4 x[T][4];
#pragma unroll
        for (int t = 0; t < T; ++t)
#pragma unroll
            for (int s = 0; s < 4; ++s) x[t][s] = *reinterpret_cast<const U32x4*>(x_row[t] + 256 * block + 64 * s);
#pragma unroll
        for (int h = 0; h < kPer; ++h) {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                F32x4 sum[T];
#pragma unroll
                for (int t = 0; t < T; ++t) sum[t] = F32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < kGroupSteps; ++s) {
                    const U32x4 a = codes_bf16(b.words[j][h * kGroupSteps + s]);
#pragma unroll
                    for (int t = 0; t < T; ++t) sum[t] = mfma(a, x[t][h * kGroupSteps + s], sum[t]);
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
    // (The host sends larger x to linear_int4_plain_kernel.)
    const int copy_rows = rows > 4 ? 8 : rows > 2 ? 4 : rows;  // rows that the waves copy at a time
    const __amdgpu_buffer_rsrc_t x_all = handoff_resource(p.x, (uint32_t)(((p.rows - 1) * p.x_stride + p.in_features) * 2));
    for (int first = 0; first < blocks; first += p.chunk_blocks) {
        const int count = min(p.chunk_blocks, blocks - first);
        const int begin = first + count * part / WK, end = first + count * (part + 1) / WK;
        // (Loads without a condition, past the end of the last block again: after a
        // load that one path leaves out, every wait is for all loads in flight.)
        Codes codes[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) load_codes(codes[a], min(begin + a, blocks - 1));
        if (first > 0) __syncthreads();
        // 1 KB of a row per DMA load, all in flight; zeros past the inputs.
        const int pieces = (count + 3) / 4;
        for (int r = wave & (copy_rows - 1); r < rows; r += copy_rows) {
            const uint32_t row = (uint32_t)(r * p.x_stride + 128 * first) * 2;
            uint8_t* to = lds + r * row_bytes;
            for (int c = wave / copy_rows; c < pieces; c += 8 / copy_rows) {
                const int at = 512 * c + 8 * lane;  // of the chunk
                load_to_lds(x_all, to + 1024 * c, 128 * first + at < in_features ? row + 2 * at : 0xfffffff0u);
            }
        }
        wait_vector_memory();
        __syncthreads();
        for (int b = begin; b < end; b += kAhead) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (b + a < end) compute(codes[a], b + a - first);
                load_codes(codes[a], min(b + a + kAhead, blocks - 1));
            }
        }
    }

    // ---------------------------------------------------------------- join
    auto write = [&](F32x4 sum, int64_t tile, int t) {
        const int64_t n = 16 * tile + 4 * g, m = 16 * t + i;
        if (m >= p.rows) return;
        if (p.aligned && n + 4 <= p.out_features) {
            *reinterpret_cast<uint2*>(p.y + m * p.y_stride + n) =
                make_uint2(bf16x2_rn(kCodeUnit * sum[0], kCodeUnit * sum[1]), bf16x2_rn(kCodeUnit * sum[2], kCodeUnit * sum[3]));
            return;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (n + r >= p.out_features) break;
            p.y[m * p.y_stride + n + r] = (uint16_t)bf16_rn(kCodeUnit * sum[r]);
        }
    };
    if constexpr (WK == 1) {
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int t = 0; t < T; ++t) write(total[j][t], tile0 + j, t);
    } else {
        F32x4(*const partial)[NB * T][64] = reinterpret_cast<F32x4(*)[NB * T][64]>(lds);  // [wave][output][lane]
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int t = 0; t < T; ++t) partial[wave][j * T + t][lane] = total[j][t];
        __syncthreads();
        // The waves of a group of tiles share its outputs out.
        for (int q = part; q < NB * T; q += WK) {
            F32x4 sum = partial[wave - part][q][lane];
#pragma unroll
            for (int w = 1; w < WK; ++w) sum += partial[wave - part + w][q][lane];
            write(sum, tile0 + q / T, q % T);
        }
    }
}

// One workgroup of W waves per tile of 16 outputs and 16 rows: x goes from
// global memory to the operands without LDS, which saves few rows a copy and a
// barrier.  All of a wave's blocks, at most kBlocks, are in flight at once;
// past its last one a wave reads that block again and leaves its sums out (a branch
// around it would let the compiler move its loads behind the first block's products).
template <int Group, int kBlocks, int W>
__global__ __launch_bounds__(64 * W) void linear_int4_few_kernel(const LinearInt4Params p) {
    constexpr int kPer = 128 / Group, kGroupSteps = Group / 32;
    __shared__ F32x4 partial[W][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int in_features = (int)p.in_features, blocks = (int)int4_blocks(p.in_features);
    const int64_t tile = blockIdx.x, first_row = 16 * blockIdx.y;
    const int rows = min((int)(p.rows - first_row), 16);
    const int begin = blocks * wave / W, end = blocks * (wave + 1) / W;
    const uint16_t* x_row = p.x + (first_row + min(i, rows - 1)) * p.x_stride + 8 * g;
    U32x4 words[kBlocks], x[kBlocks][4];
    uint32_t scales[kBlocks][2 * kPer];
#pragma unroll
    for (int a = 0; a < kBlocks; ++a) {
        const int block = min(min(begin + a, end - 1), blocks - 1);
        const int64_t place = tile * blocks + max(block, 0);
        words[a] = __builtin_nontemporal_load(reinterpret_cast<const U32x4*>(p.packed) + place * 64 + lane);
        const uint32_t* from = reinterpret_cast<const uint32_t*>(p.packed_scales) + place * (8 * kPer) + g * (2 * kPer);
#pragma unroll
        for (int h = 0; h < kPer; ++h) {
            const uint2 v = reinterpret_cast<const uint2*>(from)[h];
            scales[a][2 * h] = v.x;
            scales[a][2 * h + 1] = v.y;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = 128 * max(block, 0) + 32 * s;
            x[a][s] = *reinterpret_cast<const U32x4*>(x_row + (k < in_features ? k : 0));
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    F32x4 total = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int a = 0; a < kBlocks; ++a) {
        F32x4 sum[kPer];
#pragma unroll
        for (int h = 0; h < kPer; ++h) sum[h] = F32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < kGroupSteps; ++s)
#pragma unroll
            for (int h = 0; h < kPer; ++h)
                sum[h] = mfma(codes_bf16(words[a][h * kGroupSteps + s]), x[a][h * kGroupSteps + s], sum[h]);
#pragma unroll
        for (int h = 0; h < kPer; ++h) {
            const float scale[4] = {__uint_as_float(scales[a][2 * h] << 16), __uint_as_float(scales[a][2 * h] & 0xffff0000u),
                                    __uint_as_float(scales[a][2 * h + 1] << 16), __uint_as_float(scales[a][2 * h + 1] & 0xffff0000u)};
            // (What was read again may hold infinities: no sum of it counts, not even times 0.)
            const bool counts = begin + a < end && 128 * (begin + a) + Group * h < in_features;
#pragma unroll
            for (int r = 0; r < 4; ++r) total[r] = counts ? fmaf(scale[r], sum[h][r], total[r]) : total[r];
        }
    }
    partial[wave][lane] = total;
    __syncthreads();
    if (wave == 0 && i < rows) {
#pragma unroll
        for (int w = 1; w < W; ++w) total += partial[w][lane];
        const int64_t n = 16 * tile + 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (n + r >= p.out_features) break;
            p.y[(first_row + i) * p.y_stride + n + r] = (uint16_t)bf16_rn(kCodeUnit * total[r]);
        }
    }
}

// One workgroup per tile of 16 outputs, in plain steps: rows of x too far
// apart for the others' addresses.
__global__ __launch_bounds__(256) void linear_int4_plain_kernel(const LinearInt4Params p) {
    const int64_t blocks = int4_blocks(p.in_features), tile = blockIdx.x;
    for (int o = threadIdx.x; o < 16 * (int)p.rows; o += 256) {
        const int64_t n = 16 * tile + o % 16, m = o / 16;
        if (n >= p.out_features) continue;
        float sum = 0.f;
        for (int64_t k = 0; k < p.in_features; k += 8) {
            const uint32_t word = p.packed[((tile * blocks + k / 128) * 64 + (n & 15) + 16 * (k / 8 % 4)) * 4 + k / 32 % 4];
            const float scale = bf16_f32(p.packed_scales[scale_place(tile, blocks, k / p.group, p.group, (int)(n & 15))]);
            for (int e = 0; e < 8; ++e)
                sum = fmaf(scale, (float)code_at(word, e) / kCodeUnit * bf16_f32(p.x[m * p.x_stride + k + e]), sum);
        }
        p.y[m * p.y_stride + n] = (uint16_t)bf16_rn(kCodeUnit * sum);
    }
}

template <int Group, int T, int NB, int WK>
void launch_one(const LinearInt4Params& p, size_t bytes, hipStream_t stream) {
    const int64_t per = 8 / WK * NB, tiles = int4_tiles(p.out_features);
    hipLaunchKernelGGL((linear_int4_kernel<Group, T, NB, WK>), dim3((unsigned)((tiles + per - 1) / per)),
                       dim3(kLinearInt4Threads), std::max<size_t>(bytes, 8 * NB * T * 1024), stream, p);
}

template <int Group, int Blocks, int W>
void launch_few(const LinearInt4Params& p, hipStream_t stream) {
    const dim3 grid((unsigned)int4_tiles(p.out_features), (unsigned)((p.rows + 15) / 16));
    hipLaunchKernelGGL((linear_int4_few_kernel<Group, Blocks, W>), grid, dim3(64 * W), 0, stream, p);
}

template <int Group, int T>
void launch_tiles(const LinearInt4Params& p, hipStream_t stream) {
    const int64_t tiles = int4_tiles(p.out_features);
    const int blocks = (int)int4_blocks(p.in_features);
    LinearInt4Params q = p;
    q.aligned = p.y_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.y) % 8 == 0;
    // x of one chunk in LDS: all of it up to 152 KB, else chunks of at most that.
    auto chunk_bytes = [&](int64_t count) { return p.rows * ((count + 3) / 4 * 1024 + kRowPad); };
    q.chunk_blocks = blocks;
    while (chunk_bytes(q.chunk_blocks) > 152 * 1024) q.chunk_blocks = (q.chunk_blocks - 1) / 4 * 4;  // (whole KB of a row)
    const size_t bytes = chunk_bytes(q.chunk_blocks);
    // Tiles per workgroup: every compute unit takes ceil(workgroups / units)
    // workgroups, each a copy of x (at 125 KB per us) and its tiles (21 KB of
    // codes per us and compute unit, the even share of the memory's rate).
    const double copy = p.rows * (double)blocks * 256 / 125e3 + 0.5, tile = blocks * 1024 / 21e3;
    constexpr int kChoices[6][3] = {{1, 1, 8}, {2, 2, 8}, {3, 3, 8}, {4, 1, 2}, {8, 2, 2}, {12, 3, 2}};  // tiles, NB, WK
    int best = 0;
    double least = 0;
    for (int c = 0; c < 6; ++c) {
        const int64_t workgroups = (tiles + kChoices[c][0] - 1) / kChoices[c][0];
        const double time = (double)((workgroups + q.compute_units - 1) / q.compute_units) * (copy + kChoices[c][0] * tile);
        if (c == 0 || time < least) best = c, least = time;
    }
    switch (best) {
        case 0: return launch_one<Group, T, 1, 8>(q, bytes, stream);
        case 1: return launch_one<Group, T, 2, 8>(q, bytes, stream);
        case 2: return launch_one<Group, T, 3, 8>(q, bytes, stream);
        case 3: return launch_one<Group, T, 1, 2>(q, bytes, stream);
        case 4: return launch_one<Group, T, 2, 2>(q, bytes, stream);
        default: return launch_one<Group, T, 3, 2>(q, bytes, stream);
    }
}

// x beside the codes, or through LDS: by the rounds of workgroups, one per tile
// and 16 rows, that the compute units take without it.  Without LDS (against
// with it), for outputs x inputs and rows:
//   1 round:   2048 x 5632, 16: 8.7 us (8.5); 32: 9.0 (11.3)
//   2 rounds:  2048 x 5632, 64: 16.0 us (20.1); 4096 x 5632, 32: 16.0 (12.2)
//   3 rounds:  11264 x 2048, 8: 7.2 us (7.4), 16: 9.2 (7.8); 12288 x 1024, 16: 6.0 (6.5); 6144 x 1024, 32: 6.0 (5.7)
//   4 rounds:  16000 x 2048, 8: 8.5 us (7.4); 4096 x 1024, 64: 7.1 (5.9)
// and with 4 waves: 6144 x 512, 16 (2 rounds): 3.5 us (4.3); 16000 x 512, 16 (4): 4.9 (4.8); 11264 x 512, 32 (6): 6.1
// (5.9); 16000 x 512, 32 (8): 7.1 (5.2).
template <int Group>
void launch_rows(const LinearInt4Params& p, hipStream_t stream) {
    const int blocks = (int)int4_blocks(p.in_features);
    const int64_t workgroups = int4_tiles(p.out_features) * ((p.rows + 15) / 16);
    const int64_t rounds = (workgroups + p.compute_units - 1) / p.compute_units;
    const int64_t most = blocks <= 4 ? 6 : blocks <= 8 || (blocks <= 24 && p.rows <= 8) ? 3 : p.rows > 32 ? 2 : 1;
    if (blocks <= 48 && rounds <= most) {
        // (Four waves where they hold all inputs: 6144 x 512, 16 rows 3.5 us against 4.5 with eight, which
        // at 1024 inputs take 4.6 against 4.8; sixteen past 24 blocks, for one row: 2048 x 5632 5.6 us against
        // 5.8, 2048 x 4096 4.6 against 4.5; with 16 rows 8.8 against 8.6 and 6.6 against 6.5.)
        if (blocks <= 4)
            launch_few<Group, 1, 4>(p, stream);
        else if (blocks <= 8)
            launch_few<Group, 1, 8>(p, stream);
        else if (blocks <= 16)
            launch_few<Group, 2, 8>(p, stream);
        else if (blocks <= 24)
            launch_few<Group, 3, 8>(p, stream);
        else if (blocks <= 32)
            launch_few<Group, 2, 16>(p, stream);
        else
            launch_few<Group, 3, 16>(p, stream);
        return;
    }
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
    if (p.x_stride >= (1 << 24))  // 64 rows would pass the 2 GiB that the DMA loads of x address
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
