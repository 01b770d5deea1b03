// Verification of drafted tokens.  Row r of a request holds the distribution p_r
// of the token behind token t_r; all rows but the last have a draft t_{r+1},
// drawn from q_r.  With given random numbers u_r the draft is taken iff
// u_r q_r(t_{r+1}) < p_r(t_{r+1}); the first row whose draft is not, or the last
// row, is the final one.  Its token is drawn from the weights
// w = max(p - q, 0) (p in the last row) with the last row's u: the lowest token
// with w > 0 whose cumulative sum exceeds u times the whole.
//
// Sums are FP64: in FP32 their rounding, some 10^-7 of the whole, would move one
// border in thirty among 150000 tokens past a given u; in FP64 none.
#include <algorithm>

#include "rq_device.h"
#include "rq_reduced.h"

namespace rq {

namespace {

constexpr int kVerifyThreads = 256;

template <bool Bf16>
__device__ __forceinline__ double probability_at(const void* row, int64_t i) {
    const float p = Bf16 ? bf16_f32(static_cast<const uint16_t*>(row)[i]) : static_cast<const float*>(row)[i];
    // What is no probability counts as 0.
    return p > 0.f && p < __builtin_inff() ? (double)p : 0.0;
}

// A request's rows, and the final one of them.
struct VerifyRequest {
    int64_t first, stop, end;
};

template <bool Bf16>
__device__ __forceinline__ const void* row_of(const void* base, int64_t stride, int64_t row) {
    return static_cast<const uint8_t*>(base) + row * stride * (Bf16 ? 2 : 4);
}

// (Every wave finds the final row by itself.)
template <bool Bf16>
__device__ __forceinline__ VerifyRequest verify_request(const VerifyParams& p, int64_t request) {
    VerifyRequest r;
    r.first = p.query_start_loc[request];
    r.stop = min((int64_t)p.query_start_loc[request + 1], p.rows);
    if (r.first < 0 || r.first > r.stop) r.stop = r.first = max((int64_t)0, min(r.first, p.rows));
    r.end = r.stop - 1;
    const int lane = threadIdx.x & 63;
    for (int64_t base = r.first; base < r.stop - 1; base += 64) {
        const int64_t row = base + lane;
        bool refused = false;
        if (row < r.stop - 1) {
            const int64_t token = p.tokens[row + 1];
            double of_target = 0.0, of_draft = 1.0;
            if (token >= 0 && token < p.vocab) {
                of_target = probability_at<Bf16>(row_of<Bf16>(p.target, p.target_stride, row), token);
                if (p.draft != nullptr) of_draft = probability_at<Bf16>(row_of<Bf16>(p.draft, p.draft_stride, row), token);
            }
            refused = !((double)p.uniforms[row] * of_draft < of_target);
        }
        const uint64_t found = __ballot(refused);
        if (found != 0) {
            r.end = base + __builtin_ctzll(found);
            break;
        }
    }
    return r;
}

// The weights of a final row.
template <bool Bf16>
struct Weights {
    const void* target;
    const void* draft;  // null: nothing is taken off
    int64_t without;    // a token that does not count
    __device__ Weights(const VerifyParams& p, const VerifyRequest& r) {
        const bool refused = r.end < r.stop - 1;
        target = row_of<Bf16>(p.target, p.target_stride, r.end);
        draft = refused && p.draft != nullptr ? row_of<Bf16>(p.draft, p.draft_stride, r.end) : nullptr;
        without = refused && p.draft == nullptr ? p.tokens[r.end + 1] : -1;
    }
    __device__ __forceinline__ double at(int64_t token) const {
        double w = probability_at<Bf16>(target, token);
        if (draft != nullptr) w = fmax(w - probability_at<Bf16>(draft, token), 0.0);
        return token == without ? 0.0 : w;
    }
};

__device__ __forceinline__ double shuffle_xor_f64(double v, int d) { return __shfl_xor(v, d); }

// The sum of the workgroup's values, in every thread.
__device__ __forceinline__ double block_sum(double v, double* partial) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += shuffle_xor_f64(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = v;
    __syncthreads();
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < kVerifyThreads / 64; ++w) total += partial[w];
    return total;
}

// One workgroup per chunk of a request's final row: the sum of its weights.
template <bool Bf16>
__global__ __launch_bounds__(kVerifyThreads) void verify_sums_kernel(const VerifyParams p) {
    __shared__ double partial[kVerifyThreads / 64];
    const int64_t request = blockIdx.x / p.chunks, chunk = blockIdx.x % p.chunks;
    const VerifyRequest r = verify_request<Bf16>(p, request);
    if (r.first == r.stop) return;
    const Weights<Bf16> weights(p, r);
    const int64_t begin = chunk * p.chunk, end = min(begin + p.chunk, p.vocab);
    double sum = 0.0;
    for (int64_t t = begin + threadIdx.x; t < end; t += kVerifyThreads) sum += weights.at(t);
    sum = block_sum(sum, partial);
    if (threadIdx.x == 0) p.sums[request * p.chunks + chunk] = sum;
}

// The first of `count` values whose running sum, from `before` on, exceeds
// `limit` and that is above 0 itself, else the last above 0, else -1; and the
// running sum before it.  For a wave; value(k) gives the k-th.
struct Found {
    int64_t place;
    double before;
};
template <class Value>
__device__ __forceinline__ Found find_above(int64_t count, double before, double limit, Value value) {
    const int lane = threadIdx.x & 63;
    Found last{-1, before};
    for (int64_t base = 0; base < count; base += 64) {
        const double own = base + lane < count ? value(base + lane) : 0.0;
        double running = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const double below = __shfl_up(running, d);
            if (lane >= d) running += below;
        }
        const uint64_t any = __ballot(own > 0.0), above = __ballot(own > 0.0 && before + running > limit);
        const uint64_t pick = above != 0 ? above & -above : any;
        if (pick != 0) {
            const int at = 63 - __builtin_clzll(pick);
            last = Found{base + at, before + __shfl(running - own, at)};
            if (above != 0) return last;
        }
        before += __shfl(running, 63);
    }
    return last;
}

// One wave per request.
template <bool Bf16>
__global__ __launch_bounds__(64) void verify_draw_kernel(const VerifyParams p) {
    const int64_t request = blockIdx.x;
    const int lane = threadIdx.x;
    const VerifyRequest r = verify_request<Bf16>(p, request);
    // Rows outside of every request have no token.
    if (request == 0)
        for (int64_t row = lane; row < r.first; row += 64) p.out_tokens[row] = -1;
    if (request == p.requests - 1)
        for (int64_t row = r.stop + lane; row < p.rows; row += 64) p.out_tokens[row] = -1;
    if (lane == 0) p.accepted[request] = r.first == r.stop ? 0 : (int32_t)(r.end - r.first);
    if (r.first == r.stop) return;
    const Weights<Bf16> weights(p, r);
    const double* sums = p.sums + request * p.chunks;
    double whole = 0.0;
    for (int64_t c = lane; c < p.chunks; c += 64) whole += sums[c];
#pragma unroll
    for (int d = 32; d; d >>= 1) whole += shuffle_xor_f64(whole, d);
    const double limit = (double)p.uniforms[r.stop - 1] * whole;
    const Found chunk = find_above(p.chunks, 0.0, limit, [&](int64_t c) { return sums[c]; });
    int64_t token = -1;
    if (chunk.place >= 0) {
        const int64_t begin = chunk.place * p.chunk;
        token = find_above(min(p.chunk, p.vocab - begin), chunk.before, limit,
                           [&](int64_t t) { return weights.at(begin + t); }).place;
        if (token >= 0) token += begin;
    }
    for (int64_t row = r.first + lane; row < r.stop; row += 64)
        p.out_tokens[row] = row < r.end ? p.tokens[row + 1] : row == r.end ? token : -1;
}

template <bool Bf16>
void launch(const VerifyParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(verify_sums_kernel<Bf16>, dim3((unsigned)(p.requests * p.chunks)), dim3(kVerifyThreads), 0, stream, p);
    hipLaunchKernelGGL(verify_draw_kernel<Bf16>, dim3((unsigned)p.requests), dim3(64), 0, stream, p);
}

}  // namespace

// Tokens per workgroup: a row's chunks, in whole rounds of the threads.
int64_t verify_chunks(int64_t requests, int64_t vocab, int64_t* chunk) {
    (void)requests;
    *chunk = 2048;
    return (vocab + *chunk - 1) / *chunk;
}

hipError_t launch_verify(const VerifyParams& p, hipStream_t stream) {
    if (p.bf16)
        launch<true>(p, stream);
    else
        launch<false>(p, stream);
    return hipGetLastError();
}

}  // namespace rq
