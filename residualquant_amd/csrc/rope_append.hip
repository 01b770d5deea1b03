// Fused [q | k | v] rows of a call's new tokens: q and k rotated to their
// positions (pairs (a, b) of the first `rotary` channels become
// (a cos - b sin, b cos + a sin), halves of the rotated channels or neighbours),
// and k and v appended to a paged cache on the way: E4M3 pages with one
// power-of-two scale per (plane, block, head), as quantize_fp8_kernel writes
// them, or BF16 pages.
//
// Bytes bound it: each row is read once and written twice (k and v also to
// their pages).  One wave per (page that the call writes, head, plane), planes K,
// V and Q: a page's new values stay in registers between their maximum and
// their conversion.  Request b's pages take the slots from
// floor(first row / PT) + 2 b (n rows touch at most n / PT + 2 pages), so a wave
// finds its request by counting.
#include "rq_device.h"
#include "rq_fp8.h"
#include "rq_reduced.h"

namespace rq {

namespace {

typedef float F32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void unpack(U32x4 raw, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = __uint_as_float(raw[e] << 16);
        x[2 * e + 1] = __uint_as_float(raw[e] & 0xffff0000u);
    }
}
__device__ __forceinline__ U32x4 pack(const float (&x)[8]) {
    return U32x4{bf16x2_rn(x[0], x[1]), bf16x2_rn(x[2], x[3]), bf16x2_rn(x[4], x[5]), bf16x2_rn(x[6], x[7])};
}

// Both products and their sum are rounded (no fma), so that a pair's two channels round alike.
__device__ __forceinline__ float minus(float a, float c, float b, float s) {
#pragma clang fp contract(off)
    return a * c - b * s;
}
__device__ __forceinline__ float plus(float a, float c, float b, float s) {
#pragma clang fp contract(off)
    return a * c + b * s;
}

// Channels 8 column.. of a row's head at `x`, rotated.
__device__ __forceinline__ U32x4 rotated(const RopeAppendParams& p, const uint16_t* x, int column, int64_t position) {
    const U32x4 own_raw = *reinterpret_cast<const U32x4At8*>(x + 8 * column);
    const int channel = 8 * column, half = p.rotary / 2;
    if (channel >= p.rotary) return own_raw;
    float own[8], out[8];
    unpack(own_raw, own);
    if (p.interleaved) {
        const F32x4 c = *reinterpret_cast<const F32x4*>(p.cos_table + position * half + channel / 2);
        const F32x4 s = *reinterpret_cast<const F32x4*>(p.sin_table + position * half + channel / 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            out[2 * e] = minus(own[2 * e], c[e], own[2 * e + 1], s[e]);
            out[2 * e + 1] = plus(own[2 * e + 1], c[e], own[2 * e], s[e]);
        }
        return pack(out);
    }
    const bool first = channel < half;
    const int at = first ? channel : channel - half;
    float other[8];
    unpack(*reinterpret_cast<const U32x4At8*>(x + (first ? channel + half : at)), other);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const F32x4 c = *reinterpret_cast<const F32x4*>(p.cos_table + position * half + at + 4 * h);
        const F32x4 s = *reinterpret_cast<const F32x4*>(p.sin_table + position * half + at + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            out[4 * h + e] = first ? minus(own[4 * h + e], c[e], other[4 * h + e], s[e])
                                   : plus(own[4 * h + e], c[e], other[4 * h + e], s[e]);
    }
    return pack(out);
}

enum { kPlaneKey = 0, kPlaneValue = 1, kPlaneQuery = 2 };

template <int D, int PT, bool Fp8>
__global__ __launch_bounds__(256) void rope_append_kernel(const RopeAppendParams p) {
    constexpr int kRow = D / 8;                      // chunks of 8 values per row
    constexpr int kChunks = kPageChunks<D, PT>;
    constexpr int kShift = PT == 16 ? 4 : 5;
    const int lane = threadIdx.x & 63;
    const int head = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int plane = blockIdx.z;
    if (head >= (plane == kPlaneQuery ? p.heads : p.kv_heads)) return;
    const int request = write_request(p.query_start_loc, (int)p.requests, kShift, (int)blockIdx.x);
    const int first = p.query_start_loc[request];
    const int n = p.query_start_loc[request + 1] - first;
    const int64_t seq = p.seq_lens[request];
    const int64_t history = seq > n ? seq - n : 0;
    // The page: the slot's number among the request's, the rows from `begin` on at `slot`.
    const int64_t number = (int64_t)blockIdx.x - ((int64_t)(first >> kShift) + 2 * (int64_t)request);
    const int64_t page = (history >> kShift) + number;
    const int64_t begin = number == 0 ? 0 : (page << kShift) - history;
    if (n <= 0 || first < 0 || number < 0 || begin >= n || first + begin >= p.rows) return;
    const int slot = (int)((history + begin) & (PT - 1));
    const int rows = (int)min(min((int64_t)(PT - slot), n - begin), p.rows - first - begin);
    const int64_t row0 = first + begin;
    const int in_head = plane == kPlaneQuery ? head : p.heads + plane * p.kv_heads + head;
    const uint16_t* in = p.qkv + row0 * p.qkv_stride + (int64_t)in_head * D;

    U32x4 values[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int chunk = 64 * c + lane, r = chunk / kRow, column = chunk - r * kRow;
        values[c] = U32x4{0u, 0u, 0u, 0u};
        if (r >= rows) continue;
        const uint16_t* x = in + r * p.qkv_stride;
        if (plane == kPlaneValue) {
            values[c] = *reinterpret_cast<const U32x4At8*>(x + 8 * column);
            continue;
        }
        const int64_t given = p.positions != nullptr ? p.positions[row0 + r] : history + begin + r;
        values[c] = rotated(p, x, column, min(max(given, (int64_t)0), p.table_rows - 1));
        uint16_t* out = plane == kPlaneQuery ? p.query + (row0 + r) * p.query_stride : p.key + (row0 + r) * p.key_stride;
        *reinterpret_cast<U32x4At8*>(out + (int64_t)head * D + 8 * column) = values[c];
    }
    if (plane == kPlaneQuery || page >= p.max_pages) return;
    const int64_t block = p.block_table[(int64_t)request * p.block_table_stride + page];
    if (block < 0 || block >= p.num_blocks) return;
    const int64_t index = ((int64_t)plane * p.num_blocks + block) * p.kv_heads + head;

    if constexpr (!Fp8) {
        U32x4* const to = reinterpret_cast<U32x4*>(static_cast<uint16_t*>(p.cache) + index * (PT * D)) + slot * kRow;
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
            if (64 * c + lane < rows * kRow) to[64 * c + lane] = values[c];
        return;
    }
    float* const scale = p.scales + index;
    write_fp8_page<D, PT>(values, static_cast<uint8_t*>(p.cache) + index * (PT * D), scale, *scale, slot, rows);
}

template <int D, int PT>
void launch_pages(const RopeAppendParams& p, hipStream_t stream) {
    const int64_t slots = p.rows / PT + 2 * p.requests;
    const dim3 grid((unsigned)slots, (unsigned)((max(p.heads, p.kv_heads) + 3) / 4), 3);
    if (p.scales != nullptr)
        hipLaunchKernelGGL((rope_append_kernel<D, PT, true>), grid, dim3(256), 0, stream, p);
    else
        hipLaunchKernelGGL((rope_append_kernel<D, PT, false>), grid, dim3(256), 0, stream, p);
}

}  // namespace

hipError_t launch_rope_append(const RopeAppendParams& p, hipStream_t stream) {
    if (p.head_dim == 128)
        p.page_tokens == 16 ? launch_pages<128, 16>(p, stream) : launch_pages<128, 32>(p, stream);
    else
        p.page_tokens == 16 ? launch_pages<96, 16>(p, stream) : launch_pages<96, 32>(p, stream);
    return hipGetLastError();
}

}  // namespace rq
