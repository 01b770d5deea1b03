// Log probability of given tokens, entropy and top alternatives of logits:
// with m = max x and S = sum e^(x - m), log p = x - m - log S and
// H = log S - sum e^(x - m) (x - m) / S, where entries of -inf add nothing.
#include "rq_device.h"
#include "rq_reduced.h"

namespace rq {

namespace {

constexpr int kLogprobThreads = 256;

template <bool Bf16>
__device__ __forceinline__ float logit_at(const void* logits, int64_t i) {
    if constexpr (Bf16)
        return bf16_f32(static_cast<const uint16_t*>(logits)[i]);
    else
        return static_cast<const float*>(logits)[i];
}

// Order of (value, index) as one number: greater values first, equal ones
// (-0 and +0 among them) by the lower index, NaN above all.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    const uint32_t ordered = x != x ? 0xffffffffu : (u >> 31) ? ~u : u | 0x80000000u;
    return ((uint64_t)ordered << 32) | (0xffffffffu - index);
}

__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* partial) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint64_t other = ((uint64_t)__shfl_xor((uint32_t)(v >> 32), d) << 32) | __shfl_xor((uint32_t)v, d);
        v = other > v ? other : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < kLogprobThreads / 64; ++w) v = partial[w] > v ? partial[w] : v;
    return v;
}

__device__ __forceinline__ float block_sum(float v, float* partial) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = v;
    __syncthreads();
    float total = 0.f;
    for (int w = 0; w < kLogprobThreads / 64; ++w) total += partial[w];
    return total;
}

// One workgroup per row: one pass for the maximum, one for the sums, one for
// each alternative.
template <bool Bf16>
__global__ __launch_bounds__(kLogprobThreads) void logprobs_kernel(const LogprobParams p) {
    __shared__ uint64_t keys[kLogprobThreads / 64];
    __shared__ float sums[kLogprobThreads / 64];
    const int64_t row = blockIdx.x;
    const int64_t base = row * p.stride;
    float largest = -__builtin_inff();
    for (int64_t i = threadIdx.x; i < p.vocab; i += kLogprobThreads) largest = fmaxf(largest, logit_at<Bf16>(p.logits, base + i));
    const uint64_t top_key = block_max_u64(rank_key(largest, 0), keys);
    const uint32_t ordered = (uint32_t)(top_key >> 32);
    largest = __uint_as_float((ordered >> 31) ? ordered & 0x7fffffffu : ~ordered);
    float sum = 0.f, weighted = 0.f;
    for (int64_t i = threadIdx.x; i < p.vocab; i += kLogprobThreads) {
        const float x = logit_at<Bf16>(p.logits, base + i);
        const float d = x - largest, w = x == -__builtin_inff() ? 0.f : expf(d);
        sum += w;
        weighted += w > 0.f ? w * d : 0.f;
    }
    sum = block_sum(sum, sums);
    weighted = block_sum(weighted, sums);
    const float log_sum = logf(sum);
    if (threadIdx.x == 0) {
        const int64_t token = p.tokens[row];
        p.logprob[row] = token >= 0 && token < p.vocab ? logit_at<Bf16>(p.logits, base + token) - largest - log_sum
                                                       : __builtin_nanf("");
        p.entropy[row] = log_sum - weighted / sum;
    }
    uint64_t below = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        uint64_t best = 0;
        for (int64_t i = threadIdx.x; i < p.vocab; i += kLogprobThreads) {
            const uint64_t key = rank_key(logit_at<Bf16>(p.logits, base + i), (uint32_t)i);
            if (key < below && key > best) best = key;
        }
        below = best = block_max_u64(best, keys);
        if (threadIdx.x == 0) {
            const int64_t index = 0xffffffffu - (uint32_t)best;
            p.top_tokens[row * p.top + k] = index;
            p.top_logprobs[row * p.top + k] = logit_at<Bf16>(p.logits, base + index) - largest - log_sum;
        }
    }
}

}  // namespace

hipError_t launch_logprobs(const LogprobParams& p, hipStream_t stream) {
    if (p.bf16)
        hipLaunchKernelGGL((logprobs_kernel<true>), dim3((unsigned)p.rows), dim3(kLogprobThreads), 0, stream, p);
    else
        hipLaunchKernelGGL((logprobs_kernel<false>), dim3((unsigned)p.rows), dim3(kLogprobThreads), 0, stream, p);
    return hipGetLastError();
}

}  // namespace rq
