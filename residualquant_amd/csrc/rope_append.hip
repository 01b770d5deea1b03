// Fused [q | k | v] rows of a call's new tokens: q and k rotated to their
// positions (pairs (a, b) of the first `rotary` channels become
// (a cos - b sin, b cos + a sin), halves of the rotated channels or neighbours),
// and k and v appended to a paged cache on the way: E4M3 pages with one
// power-of-two scale per (plane, block, head), as quantize_fp8_kernel writes
// them, or BF16 pages.
//
// Bytes bound it: each row is read once and written twice (k and v also to
// their pages).  One workgroup per page that the call writes and some of its heads
// (q's, k's and v's in a row), a wave a head at a time: a page's new values stay in
// registers between their maximum and their conversion, and the angles of its rows lie
// in LDS for all of them.  A lane holds the chunks of eight channels that are turned
// together.  Request b's pages take the slots from floor(first row / PT) + 2 b (n
// rows touch at most n / PT + 2 pages), so a workgroup finds its request by counting.
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

// Chunks a < b of a row that lane slot `s` (0..D / 16 - 1) holds: the two halves of
// what is turned together, then the channels that are not turned; neighbours where
// neighbouring channels are.
__device__ __forceinline__ void chunks_of(const RopeAppendParams& p, int s, int& a, int& b) {
    const int half = p.rotary / 16;  // chunks of half of the turned channels
    const bool halves = !p.interleaved && s < half;
    a = halves ? s : 2 * s;
    b = halves ? s + half : 2 * s + 1;
}

template <int D, int PT, bool Fp8>
__global__ __launch_bounds__(256) void rope_append_kernel(const RopeAppendParams p) {
    constexpr int kRow = D / 8, kSlots = kRow / 2;   // chunks of 8 values per row, pairs of them
    constexpr int kPairs = (PT * kSlots + 63) / 64, kChunks = 2 * kPairs;  // per lane
    constexpr int kShift = PT == 16 ? 4 : 5;
    __shared__ __align__(16) float cos_of[PT * D / 2], sin_of[PT * D / 2];  // [row][rotary / 2]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    const int all_heads = p.heads + 2 * p.kv_heads;
    const int head_begin = (int)blockIdx.y * p.span, head_end = min(head_begin + p.span, all_heads);
    int64_t block = -1;
    if (head_end > p.heads && page < p.max_pages) block = p.block_table[(int64_t)request * p.block_table_stride + page];

    int at[kPairs], column[kPairs][2];  // a lane's rows (-1: none) and their chunks
#pragma unroll
    for (int c = 0; c < kPairs; ++c) {
        const int place = 64 * c + lane, r = place / kSlots;
        at[c] = r < rows ? r : -1;
        chunks_of(p, place - r * kSlots, column[c][0], column[c][1]);
    }
    U32x4 values[kChunks];
    auto load = [&](int head) {
        const uint16_t* in = p.qkv + row0 * p.qkv_stride + (int64_t)head * D;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            values[c] = U32x4{0u, 0u, 0u, 0u};
            if (at[c / 2] >= 0) values[c] = *reinterpret_cast<const U32x4At8*>(in + at[c / 2] * p.qkv_stride + 8 * column[c / 2][c & 1]);
        }
    };
    int head = head_begin + wave;
    if (head < head_end) load(head);
    const int half = p.rotary / 2;
    if (head_begin < p.heads + p.kv_heads) {
        const int quads = half / 4;
        for (int q = tid; q < rows * quads; q += 256) {
            const int r = q / quads;
            const int64_t given = p.positions != nullptr ? p.positions[row0 + r] : history + begin + r;
            const int64_t from = min(max(given, (int64_t)0), p.table_rows - 1) * half + 4 * (q - r * quads);
            *reinterpret_cast<F32x4*>(cos_of + 4 * q) = *reinterpret_cast<const F32x4*>(p.cos_table + from);
            *reinterpret_cast<F32x4*>(sin_of + 4 * q) = *reinterpret_cast<const F32x4*>(p.sin_table + from);
        }
        lds_barrier();
    }
    for (; head < head_end; head += 4) {
        if (head >= head_begin + 4) load(head);
        if (head < p.heads + p.kv_heads) {
            const bool is_query = head < p.heads;
            uint16_t* const out = is_query ? p.query + row0 * p.query_stride + (int64_t)head * D
                                           : p.key + row0 * p.key_stride + (int64_t)(head - p.heads) * D;
            const int64_t stride = is_query ? p.query_stride : p.key_stride;
#pragma unroll
            for (int c = 0; c < kPairs; ++c) {
                if (at[c] < 0) continue;
                float a[8], b[8], x[8], y[8];
                unpack(values[2 * c], a);
                unpack(values[2 * c + 1], b);
                const float* const cos_row = cos_of + at[c] * half;
                const float* const sin_row = sin_of + at[c] * half;
                if (8 * column[c][0] >= p.rotary) {
                    // (Not turned; with neighbours turned, a pair of chunks is or is not, as their number is even.)
                } else if (p.interleaved) {
                    const F32x4 cs[2] = {*reinterpret_cast<const F32x4*>(cos_row + 4 * column[c][0]), *reinterpret_cast<const F32x4*>(cos_row + 4 * column[c][1])};
                    const F32x4 sn[2] = {*reinterpret_cast<const F32x4*>(sin_row + 4 * column[c][0]), *reinterpret_cast<const F32x4*>(sin_row + 4 * column[c][1])};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[2 * e] = minus(a[2 * e], cs[0][e], a[2 * e + 1], sn[0][e]);
                        x[2 * e + 1] = plus(a[2 * e + 1], cs[0][e], a[2 * e], sn[0][e]);
                        y[2 * e] = minus(b[2 * e], cs[1][e], b[2 * e + 1], sn[1][e]);
                        y[2 * e + 1] = plus(b[2 * e + 1], cs[1][e], b[2 * e], sn[1][e]);
                    }
                    values[2 * c] = pack(x);
                    values[2 * c + 1] = pack(y);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const F32x4 cs = *reinterpret_cast<const F32x4*>(cos_row + 8 * column[c][0] + 4 * h);
                        const F32x4 sn = *reinterpret_cast<const F32x4*>(sin_row + 8 * column[c][0] + 4 * h);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            x[4 * h + e] = minus(a[4 * h + e], cs[e], b[4 * h + e], sn[e]);
                            y[4 * h + e] = plus(b[4 * h + e], cs[e], a[4 * h + e], sn[e]);
                        }
                    }
                    values[2 * c] = pack(x);
                    values[2 * c + 1] = pack(y);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) *reinterpret_cast<U32x4At8*>(out + at[c] * stride + 8 * column[c][h]) = values[2 * c + h];
            }
            if (is_query) continue;
        }
        if (block < 0 || block >= p.num_blocks) continue;
        const int plane = head >= p.heads + p.kv_heads ? 1 : 0;
        const int64_t index = ((int64_t)plane * p.num_blocks + block) * p.kv_heads + (head - p.heads - plane * p.kv_heads);
        auto place = [&](int c) { return at[c / 2] < 0 ? -1 : at[c / 2] * kRow + column[c / 2][c & 1]; };
        if constexpr (Fp8) {
            float* const scale = p.scales + index;
            write_fp8_page<D, PT>(values, static_cast<uint8_t*>(p.cache) + index * (PT * D), scale, *scale, slot, place);
        } else {
            U32x4* const to = reinterpret_cast<U32x4*>(static_cast<uint16_t*>(p.cache) + index * (PT * D)) + slot * kRow;
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
                if (at[c / 2] >= 0) to[place(c)] = values[c];
        }
    }
}

// Heads per workgroup: one per wave where they are few, else two, whose angles are
// loaded once. (12 requests of 700 rows, 32 + 2 x 8 heads of 128: 44.0 us with eight heads, 43.1
// with four, 47.1 with twelve, and 66 with a wave for each head and plane that loads its
// own angles; 16 + 2 x 16 heads 37.4, 41.7 and 38.4; 32 tokens of these 5.7, 4.7 and 6.5. 12 ragged prompts
// of up to 1500 rows, 32 + 2 x 8 heads, pages of 32: 43.8 us in E4M3 and 48.1 in BF16, 4.4 to 4.5 TB/s of what
// is read and written; a large copy reaches 5.1.)
template <int D, int PT>
void launch_pages(const RopeAppendParams& given, hipStream_t stream) {
    RopeAppendParams p = given;
    const int64_t slots = p.rows / PT + 2 * p.requests;
    const int all_heads = p.heads + 2 * p.kv_heads;
    p.span = slots * ((all_heads + 3) / 4) > 2048 ? 8 : 4;
    const dim3 grid((unsigned)slots, (unsigned)((all_heads + p.span - 1) / p.span));
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
