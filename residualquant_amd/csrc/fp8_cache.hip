// Paged cache held in 8 bits: OCP E4M3 codes [2, blocks, kv_heads, PT, D] and
// one FP32 scale per (plane, block, head); a value is code * scale.
//
// quantize_fp8_kernel writes a call's new tokens, attention_fp8_kernel reads
// the cache: the 8-bit member beside the packed (2 + 4 bit) and the BF16 pages.
#include "rq_device.h"
#include "rq_reduced.h"

namespace rq {

namespace {

// ------------------------------------------------------------------ write

// The request of a row, its place among the request's new rows and its
// position in the sequence.
struct RowPlace {
    int request;      // -1: the row belongs to no request
    int index, count; // place among the request's `count` new rows
    int64_t history;  // tokens before the first of them
};

__device__ __forceinline__ RowPlace place_row(const int32_t* qsl, const int32_t* seq_lens, int64_t requests,
                                              int64_t row, int* lds_counts) {
    RowPlace r;
    r.request = find_request_parallel(qsl, requests, row, lds_counts);
    if (r.request < 0) return r;
    const int32_t begin = qsl[r.request];
    r.index = (int)(row - begin);
    r.count = qsl[r.request + 1] - begin;
    const int64_t history = (int64_t)seq_lens[r.request] - r.count;
    r.history = history > 0 ? history : 0;
    return r;
}

// The least power of two s >= 2^-126 with largest <= 448 s.  largest = m 2^e,
// 1 <= m < 2, and 448 = 1.75 * 2^8: s is 2^(e - 8), twice that where m > 1.75.
__device__ __forceinline__ float needed_scale(float largest) {
    const uint32_t u = __float_as_uint(largest);
    int exponent = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    if (exponent < 1) exponent = 1;  // 2^-126
    return __uint_as_float((uint32_t)exponent << 23);
}

// E4M3 of x; infinities, which the format lacks, become NaN.
__device__ __forceinline__ uint32_t e4m3_code(float x) {
    return fabsf(x) == __builtin_inff() ? 0x7fu : e4m3_rn(x);
}

// One workgroup per (row, head, plane); the first new row of a page writes
// all of the page's new rows and, where the scale grows, rounds the codes of
// the page's older tokens again.
__global__ __launch_bounds__(256) void quantize_fp8_kernel(const Fp8WriteParams p) {
    __shared__ int counts[4];
    __shared__ float wave_largest[4];
    const int64_t row = blockIdx.x;
    const int head = blockIdx.y, plane = blockIdx.z;
    const int tid = threadIdx.x;
    const RowPlace at = place_row(p.query_start_loc, p.seq_lens, p.requests, row, counts);
    if (at.request < 0) return;
    const int PT = p.page_tokens, D = p.head_dim;
    const int64_t position = at.history + at.index;
    const int slot = (int)(position % PT);
    const int64_t page = position / PT;
    if ((at.index != 0 && slot != 0) || page >= p.max_pages) return;
    const int64_t block = p.block_table[(int64_t)at.request * p.block_table_stride + page];
    if (block < 0 || block >= p.num_blocks) return;
    const int rows = min(PT - slot, at.count - at.index);
    const uint16_t* in = (plane == 0 ? p.key : p.value) + row * (plane == 0 ? p.key_stride : p.value_stride) +
                         (int64_t)head * D;
    const int64_t in_stride = plane == 0 ? p.key_stride : p.value_stride;
    const int64_t index = ((int64_t)plane * p.num_blocks + block) * p.kv_heads + head;
    uint8_t* codes = p.cache + index * PT * D;

    float largest = 0.f;
    for (int i = tid; i < rows * D; i += 256) {
        const float x = fabsf(bf16_f32(in[(i / D) * in_stride + i % D]));
        if (x < __builtin_inff()) largest = fmaxf(largest, x);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
    if ((tid & 63) == 0) wave_largest[tid >> 6] = largest;
    const float before = p.scales[index];
    __syncthreads();
    largest = fmaxf(fmaxf(wave_largest[0], wave_largest[1]), fmaxf(wave_largest[2], wave_largest[3]));
    const float need = needed_scale(largest);
    const float scale = slot > 0 && before >= need ? before : need;
    if (slot > 0 && scale > before) {
        const float shrink = before / scale;
        for (int i = tid; i < slot * D; i += 256) codes[i] = (uint8_t)e4m3_rn(e4m3_f32(codes[i]) * shrink);
    }
    for (int i = tid; i < rows * D; i += 256)
        codes[slot * D + i] = (uint8_t)e4m3_code(bf16_f32(in[(i / D) * in_stride + i % D]) / scale);
    if (tid == 0) p.scales[index] = scale;
}

// ------------------------------------------------------------------ attention

// One workgroup per (row, query head): each wave takes every fourth token, a
// lane two channels, with a running maximum and sum per wave.
__global__ __launch_bounds__(256) void attention_fp8_kernel(const Fp8AttentionParams p) {
    __shared__ int counts[4];
    __shared__ float merged[4][kFp8MaxDim + 2];
    const int64_t row = blockIdx.x;
    const int head = blockIdx.y, kv_head = head / (p.heads / p.kv_heads);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const RowPlace at = place_row(p.query_start_loc, p.seq_lens, p.requests, row, counts);
    if (at.request < 0) return;
    const int PT = p.page_tokens, D = p.head_dim;
    const bool active = 2 * lane < D;
    const int64_t history = min(at.history, p.max_pages * PT);
    const uint16_t* q = p.query + row * p.query_stride + (int64_t)head * D;
    float q0 = 0.f, q1 = 0.f;
    if (active) q0 = bf16_f32(q[2 * lane]) * p.softmax_scale, q1 = bf16_f32(q[2 * lane + 1]) * p.softmax_scale;
    float m = -__builtin_inff(), l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int64_t t = wave; t < history + at.index + 1; t += 4) {
        float k0 = 0.f, k1 = 0.f, v0 = 0.f, v1 = 0.f;
        if (t < history) {
            const int64_t block = p.block_table[(int64_t)at.request * p.block_table_stride + t / PT];
            if (block < 0 || block >= p.num_blocks) continue;
            const int64_t index = block * p.kv_heads + kv_head;
            const int64_t plane = p.num_blocks * p.kv_heads;
            const uint8_t* k = p.cache + (index * PT + t % PT) * D;
            const uint8_t* v = k + plane * PT * D;
            const float ks = p.scales[index], vs = p.scales[index + plane];
            if (active) {
                k0 = e4m3_f32(k[2 * lane]) * ks, k1 = e4m3_f32(k[2 * lane + 1]) * ks;
                v0 = e4m3_f32(v[2 * lane]) * vs, v1 = e4m3_f32(v[2 * lane + 1]) * vs;
            }
        } else {
            const int64_t live = row - at.index + (t - history);
            const uint16_t* k = p.key + live * p.key_stride + (int64_t)kv_head * D;
            const uint16_t* v = p.value + live * p.value_stride + (int64_t)kv_head * D;
            if (active) {
                k0 = bf16_f32(k[2 * lane]), k1 = bf16_f32(k[2 * lane + 1]);
                v0 = bf16_f32(v[2 * lane]), v1 = bf16_f32(v[2 * lane + 1]);
            }
        }
        float s = q0 * k0 + q1 * k1;
#pragma unroll
        for (int d = 32; d; d >>= 1) s += __shfl_xor(s, d);
        if (s == -__builtin_inff()) continue;
        const float next = fmaxf(m, s);
        const float keep = m == next ? 1.f : expf(m - next), weight = expf(s - next);
        l = l * keep + weight;
        o0 = o0 * keep + weight * v0;
        o1 = o1 * keep + weight * v1;
        m = next;
    }
    if (active) merged[wave][2 * lane] = o0, merged[wave][2 * lane + 1] = o1;
    if (lane == 0) merged[wave][D] = m, merged[wave][D + 1] = l;
    __syncthreads();
    if (wave != 0 || !active) return;
    float top = -__builtin_inff();
    for (int w = 0; w < 4; ++w) top = fmaxf(top, merged[w][D]);
    float total = 0.f, a = 0.f, b = 0.f;
    for (int w = 0; w < 4; ++w) {
        const float keep = merged[w][D] == top ? 1.f : expf(merged[w][D] - top);
        total += merged[w][D + 1] * keep;
        a += merged[w][2 * lane] * keep;
        b += merged[w][2 * lane + 1] * keep;
    }
    uint16_t* out = p.output + row * p.output_stride + (int64_t)head * D;
    out[2 * lane] = (uint16_t)bf16_rn(a / total);
    out[2 * lane + 1] = (uint16_t)bf16_rn(b / total);
}

}  // namespace

hipError_t launch_quantize_fp8(const Fp8WriteParams& p, hipStream_t stream) {
    if (p.rows == 0) return hipSuccess;
    hipLaunchKernelGGL(quantize_fp8_kernel, dim3((unsigned)p.rows, (unsigned)p.kv_heads, 2), dim3(256), 0, stream, p);
    return hipGetLastError();
}

hipError_t launch_attention_fp8(const Fp8AttentionParams& p, hipStream_t stream) {
    if (p.rows == 0) return hipSuccess;
    hipLaunchKernelGGL(attention_fp8_kernel, dim3((unsigned)p.rows, (unsigned)p.heads), dim3(256), 0, stream, p);
    return hipGetLastError();
}

}  // namespace rq
