// Log probability of given tokens, entropy and top alternatives of logits:
// with m = max x and S = sum e^(x - m), log p = x - m - log S and
// H = log S - sum e^(x - m) (x - m) / S, where entries of -inf add nothing.
//
// One workgroup reads a row once, in chunks of 8 logits per thread.  A thread
// keeps the sums against a reference that follows its running maximum only
// when a logit exceeds it by 5.5 (a weight of 2^8), and its largest logit with
// the chunk that holds it first.  The reference is a logit itself and is
// subtracted before the scale of e^ to 2^: one fma(x, log2(e), -reference)
// would be an instruction less per logit, but leaves the maximum of a row
// around 10^10 with e^ of the hundreds that log2(e) x is rounded by.
//
// Alternatives: the threads of one lane number form one of 64 owners.  With T
// the `top`-th largest of the owners' largest (value, chunk) - greater values
// first, then lower chunks - at least `top` logits lie at or above T, so every
// alternative does; and logits at or above T belong to threads whose own largest
// is, some 20 to 40 of them in a row in any order.  Their chunks are read again,
// by all threads, and the few logits found (at most kMaxCandidates, else the row
// takes one pass per alternative, as rows with NaN or infinities do) are ranked
// by counting.
#include <algorithm>

#include "rq_device.h"
#include "rq_plan.h"
#include "rq_rank.h"
#include "rq_reduced.h"

namespace rq {

namespace {

constexpr int kChunk = 8;
constexpr int kMaxCandidates = 2048;
constexpr float kLog2e = 1.44269504088896341f, kSlack = 5.5f;
constexpr float kLowest = -3.402823466e+38f;

template <bool Bf16>
__device__ __forceinline__ float logit_at(const void* logits, int64_t i) {
    if constexpr (Bf16)
        return bf16_f32(static_cast<const uint16_t*>(logits)[i]);
    else
        return static_cast<const float*>(logits)[i];
}

__device__ __forceinline__ uint64_t shuffle_xor_u64(uint64_t v, int d) {
    return ((uint64_t)__shfl_xor((uint32_t)(v >> 32), d) << 32) | __shfl_xor((uint32_t)v, d);
}

// A row's chunks: chunk q holds logits 8 q - shift.. of it, so that every
// chunk starts on a 16-byte boundary (32 bytes of FP32: on a 16-byte one).
template <bool Bf16>
struct Row {
    const void* base;
    int vocab, shift, chunks;
    __device__ Row(const LogprobParams& p, int64_t row) {
        base = static_cast<const uint8_t*>(p.logits) + row * p.stride * (Bf16 ? 2 : 4);
        vocab = (int)p.vocab;
        shift = (int)(reinterpret_cast<uintptr_t>(base) % 16) / (Bf16 ? 2 : 4);
        chunks = (int)(((int64_t)vocab + shift + kChunk - 1) / kChunk);
    }
    // Chunks first_whole..end_whole - 1 lie inside the row.
    __device__ __forceinline__ int first_whole() const { return shift > 0 ? 1 : 0; }
    __device__ __forceinline__ int end_whole() const { return (int)(((int64_t)vocab + shift) / kChunk); }
    // The raw words of such a chunk, and its logits.
    struct Raw {
        Chunk16 words[Bf16 ? 1 : 2];
    };
    __device__ __forceinline__ Raw load_whole(int q) const {
        Raw r;
        const Chunk16* from = reinterpret_cast<const Chunk16*>(static_cast<const uint8_t*>(base) + ((int64_t)kChunk * q - shift) * (Bf16 ? 2 : 4));
        r.words[0] = from[0];
        if constexpr (!Bf16) r.words[1] = from[1];
        return r;
    }
    __device__ __forceinline__ static void unpack(const Raw& r, float (&x)[kChunk]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (Bf16) {
                x[2 * e] = __uint_as_float(r.words[0][e] << 16);
                x[2 * e + 1] = __uint_as_float(r.words[0][e] & 0xffff0000u);
            } else {
                x[e] = __uint_as_float(r.words[0][e]);
                x[4 + e] = __uint_as_float(r.words[1][e]);
            }
        }
    }
    // Any chunk's logits; -inf outside the row.
    __device__ __forceinline__ void load(int q, float (&x)[kChunk]) const {
        const int64_t at = (int64_t)kChunk * q - shift;
        if (at >= 0 && at + kChunk <= vocab) {
            unpack(load_whole(q), x);
            return;
        }
#pragma unroll
        for (int e = 0; e < kChunk; ++e)
            x[e] = at + e >= 0 && at + e < vocab ? logit_at<Bf16>(base, at + e) : -__builtin_inff();
    }
};

// Sums of e^(x - m) and of e^(x - m) (x - m), with m = high.
struct Sums {
    float high, sum, weighted;
    // The sums against `above` >= high.  (A sum that is NaN stays; the difference may pass the range.)
    __device__ __forceinline__ void refer_to(float above) {
        const float down = high - above, keep = __builtin_amdgcn_exp2f(down * kLog2e);
        weighted = keep == 0.f ? 0.f : (weighted + sum * down) * keep;
        sum *= keep;
        high = above;
    }
};

// Sum over the wave, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
    v += __uint_as_float(plan_dpp<0xB1>(__float_as_uint(v)));   // quad_perm [1,0,3,2]
    v += __uint_as_float(plan_dpp<0x4E>(__float_as_uint(v)));   // quad_perm [2,3,0,1]
    v += __uint_as_float(plan_dpp<0x124>(__float_as_uint(v)));  // row_ror:4
    v += __uint_as_float(plan_dpp<0x128>(__float_as_uint(v)));  // row_ror:8
    const uint32_t u = __float_as_uint(v);
    return (__uint_as_float(__builtin_amdgcn_readlane(u, 0)) + __uint_as_float(__builtin_amdgcn_readlane(u, 16))) +
           (__uint_as_float(__builtin_amdgcn_readlane(u, 32)) + __uint_as_float(__builtin_amdgcn_readlane(u, 48)));
}

template <int Threads>
__device__ __forceinline__ uint64_t block_max_u64(uint64_t v, uint64_t* partial) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const uint64_t other = shuffle_xor_u64(v, d);
        v = other > v ? other : v;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < Threads / 64; ++w) v = partial[w] > v ? partial[w] : v;
    return v;
}

template <int Threads>
__device__ __forceinline__ float block_sum(float v, float* partial) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) partial[threadIdx.x >> 6] = v;
    __syncthreads();
    float total = 0.f;
    for (int w = 0; w < Threads / 64; ++w) total += partial[w];
    return total;
}

// The row by plain passes: the maximum, the sums, one pass per alternative
// (those only if `sums_done`).
template <bool Bf16, int Threads>
__device__ __noinline__ void logprobs_plain(const LogprobParams& p, int64_t row, bool sums_done, uint64_t* keys, float* sums) {
    const int64_t base = row * p.stride;
    float largest = -__builtin_inff();
    for (int64_t i = threadIdx.x; i < p.vocab; i += Threads) largest = fmaxf(largest, logit_at<Bf16>(p.logits, base + i));
    const uint32_t ordered = (uint32_t)(block_max_u64<Threads>(rank_key(largest, 0), keys) >> 32);
    largest = __uint_as_float((ordered >> 31) ? ordered & 0x7fffffffu : ~ordered);
    float sum = 0.f, weighted = 0.f;
    for (int64_t i = threadIdx.x; i < p.vocab; i += Threads) {
        const float x = logit_at<Bf16>(p.logits, base + i);
        const float d = x - largest, w = x == -__builtin_inff() ? 0.f : expf(d);
        sum += w;
        weighted += w > 0.f ? w * d : 0.f;
    }
    sum = block_sum<Threads>(sum, sums);
    weighted = block_sum<Threads>(weighted, sums);
    const float log_sum = logf(sum);
    if (threadIdx.x == 0 && !sums_done) {
        const int64_t token = p.tokens[row];
        p.logprob[row] = token >= 0 && token < p.vocab ? logit_at<Bf16>(p.logits, base + token) - largest - log_sum
                                                       : __builtin_nanf("");
        p.entropy[row] = log_sum - weighted / sum;
    }
    uint64_t below = kAboveKeys;
    for (int k = 0; k < p.top; ++k) {
        uint64_t best = 0;
        for (int64_t i = threadIdx.x; i < p.vocab; i += Threads)
            best = next_rank(best, rank_key(logit_at<Bf16>(p.logits, base + i), (uint32_t)i), below);
        below = best = block_max_u64<Threads>(best, keys);
        if (threadIdx.x == 0) {
            const int64_t index = 0xffffffffu - (uint32_t)best;
            p.top_tokens[row * p.top + k] = index;
            p.top_logprobs[row * p.top + k] = logit_at<Bf16>(p.logits, base + index) - largest - log_sum;
        }
    }
}

template <bool Bf16, int Threads>
__global__ __launch_bounds__(Threads) void logprobs_kernel(const LogprobParams p) {
    constexpr int kWaves = Threads / 64;
    __shared__ uint64_t keys[kWaves * 64];
    __shared__ float2 wave_sums[kWaves];
    __shared__ uint64_t candidates[kMaxCandidates];
    __shared__ uint16_t listed[Threads];
    __shared__ int above[64];  // owners above each
    __shared__ int listed_count, candidate_count;
    const int64_t row_number = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Row<Bf16> row(p, row_number);
    float token_logit = 0.f;
    int64_t token = 0;
    if (tid < 64) above[tid] = 0;
    if (tid == 0) {
        token = p.tokens[row_number];
        token_logit = token >= 0 && token < p.vocab ? logit_at<Bf16>(row.base, token) : __builtin_nanf("");
        listed_count = candidate_count = 0;
    }

    // One pass: the sums, and the thread's largest logit with its first chunk.
    Sums own{kLowest, 0.f, 0.f};
    float largest = -__builtin_inff();
    uint32_t largest_chunk = 0xffffffffu;
    auto take = [&](int q, const float (&x)[kChunk]) {
        const float most = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        // (The first chunk that holds it: the row's first chunk is taken last.)
        if (most > largest || largest_chunk == 0xffffffffu || (most == largest && (uint32_t)q < largest_chunk)) {
            largest_chunk = (uint32_t)q;
            largest = fmaxf(most, largest);
        }
        if (__any(most > own.high + kSlack)) own.refer_to(fmaxf(own.high, most));
#pragma unroll
        for (int e = 0; e < kChunk; ++e) {
            const float d = x[e] - own.high;
            const float w = __builtin_amdgcn_exp2f(d * kLog2e);
            own.sum += w;
            own.weighted = fmaf(w, fmaxf(d, -1000.0f), own.weighted);  // 0 where w is 0, also at d = -inf
        }
    };
    // (Loads without a condition, the next in flight while the present are summed; at the end the last again.)
    constexpr int kAhead = 4;
    const int end_whole = row.end_whole();
    int at = row.first_whole() + tid;
    if (row.first_whole() < end_whole) {
        typename Row<Bf16>::Raw now[kAhead], next[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) now[a] = row.load_whole(min(at + a * Threads, end_whole - 1));
        for (int q = row.first_whole(); q < end_whole; q += kAhead * Threads, at += kAhead * Threads) {
#pragma unroll
            for (int a = 0; a < kAhead; ++a) next[a] = row.load_whole(min(at + (kAhead + a) * Threads, end_whole - 1));
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (at + a * Threads >= end_whole) break;
                float x[kChunk];
                Row<Bf16>::unpack(now[a], x);
                take(at + a * Threads, x);
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) now[a] = next[a];
        }
    }
    // The row's ends, by the last two threads (which have the fewest chunks).
    auto edge_chunk = [&](int thread) {
        if (thread == Threads - 1 && row.first_whole() > 0) return 0;
        if (thread == Threads - 2 && end_whole < row.chunks && row.chunks - 1 >= row.first_whole()) return row.chunks - 1;
        return -1;
    };
    if (edge_chunk(tid) >= 0) {
        float x[kChunk];
        row.load(edge_chunk(tid), x);
        take(edge_chunk(tid), x);
    }
    const uint64_t own_key = ((uint64_t)ordered_bits(largest) << 32) | (0xffffffffu - largest_chunk);
    keys[tid] = own_key;
    __syncthreads();
    // The owners' largest, then the largest of all.
    uint64_t owner = keys[lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) owner = keys[64 * w + lane] > owner ? keys[64 * w + lane] : owner;
    const uint32_t ordered = wave_max_u32((uint32_t)(owner >> 32));
    const float m = __uint_as_float((ordered >> 31) ? ordered & 0x7fffffffu : ~ordered);
    own.refer_to(m);
    const float wave_total = wave_sum(own.sum), wave_weighted = wave_sum(own.weighted);
    if (lane == 0) wave_sums[wave] = make_float2(wave_total, wave_weighted);
    __syncthreads();
    float2 part = make_float2(0.f, 0.f);
    if (lane < kWaves) part = wave_sums[lane];
    const float exact_sum = wave_sum(part.x), weighted = wave_sum(part.y);
    const float log_sum = logf(exact_sum);
    // NaN, infinities, nothing but -inf: S is NaN or m is not finite.  (Else S is 1 and more.)
    if (!(fabsf(m) < __builtin_inff() && exact_sum >= 0.5f && exact_sum < 1.0e38f)) {
        __syncthreads();
        logprobs_plain<Bf16, Threads>(p, row_number, false, keys, reinterpret_cast<float*>(wave_sums));
        return;
    }
    if (tid == 0) {
        p.logprob[row_number] = token_logit - m - log_sum;
        p.entropy[row_number] = log_sum - weighted / exact_sum;
    }
    if (p.top == 0) return;

    // T: the `top`-th of the owners (the first of them every wave knows).  The waves share its comparisons out.
    uint64_t limit = ((uint64_t)ordered << 32) | wave_max_u32((uint32_t)(owner >> 32) == ordered ? (uint32_t)owner : 0u);
    auto owner_of = [&](int o) {
        return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(owner >> 32), o) << 32) |
               (uint32_t)__builtin_amdgcn_readlane((uint32_t)owner, o);
    };
    if (p.top > 1) {
        int more = 0;
#pragma unroll
        for (int k = 0; k < 64 / kWaves; ++k) {
            const int o = __builtin_amdgcn_readfirstlane(wave) * (64 / kWaves) + k;
            const uint64_t other = owner_of(o);
            more += other > owner || (other == owner && o < lane) ? 1 : 0;
        }
        if (more > 0) atomicAdd(&above[lane], more);
        __syncthreads();
        limit = owner_of(__builtin_ctzll(__ballot(above[lane] == p.top - 1)));
    }
    if (own_key >= limit && largest_chunk != 0xffffffffu) listed[atomicAdd(&listed_count, 1)] = (uint16_t)tid;
    __syncthreads();
    // A listed thread's chunks: its whole ones and, of the last two threads, the row's ends.
    const int whole = end_whole - row.first_whole(), each = (max(whole, 0) + Threads - 1) / Threads + 1;
    const int work = listed_count * each;
    for (int o = tid; o < work; o += Threads) {
        const int owner_thread = listed[o / each], number = o % each;
        int q = row.first_whole() + owner_thread + number * Threads;
        if (number == each - 1)
            q = edge_chunk(owner_thread);
        else if (q >= end_whole)
            q = -1;
        if (q < 0) continue;
        float x[kChunk];
        row.load(q, x);
#pragma unroll
        for (int e = 0; e < kChunk; ++e) {
            const int64_t index = (int64_t)kChunk * q - row.shift + e;
            const uint64_t key = ((uint64_t)ordered_bits(x[e]) << 32) | (0xffffffffu - (uint32_t)q);
            if (key >= limit && index >= 0 && index < row.vocab) {
                const int place = atomicAdd(&candidate_count, 1);
                if (place < kMaxCandidates) candidates[place] = rank_key(x[e], (uint32_t)index);
            }
        }
    }
    __syncthreads();
    const int found = candidate_count;
    if (found > kMaxCandidates) {
        logprobs_plain<Bf16, Threads>(p, row_number, true, keys, reinterpret_cast<float*>(wave_sums));
        return;
    }
    // 16 lanes count one candidate's rank.
    for (int c0 = 0; c0 < found; c0 += Threads / 16) {
        const int c = c0 + (tid >> 4);
        const uint64_t key = c < found ? candidates[c] : kAboveKeys;
        uint32_t rank = 0;
        for (int o = tid & 15; o < found; o += 16) rank += candidates[o] > key ? 1 : 0;
        rank += plan_dpp<0xB1>(rank);   // quad_perm [1,0,3,2]
        rank += plan_dpp<0x4E>(rank);   // quad_perm [2,3,0,1]
        rank += plan_dpp<0x124>(rank);  // row_ror:4
        rank += plan_dpp<0x128>(rank);  // row_ror:8
        if ((tid & 15) != 0 || c >= found || rank >= (uint32_t)p.top) continue;
        const uint32_t bits = (uint32_t)(key >> 32);
        const float x = __uint_as_float((bits >> 31) ? bits & 0x7fffffffu : ~bits);
        p.top_tokens[row_number * p.top + rank] = (int64_t)(0xffffffffu - (uint32_t)key);
        p.top_logprobs[row_number * p.top + rank] = x - m - log_sum;
    }
}

// Four waves per row for short rows, and where enough rows run beside each
// other; else eight.  (256 threads, 512, and 1024, whose start and barriers cost
// more than they share out, in us.  1 row of 8000 logits with 8 alternatives: 6.6,
// 7.3, 9.7; of 32000: 10.1, 9.4, 10.7; of 49152: 12.3, 10.7, 11.9.  600 rows of 50257
// with 1: 26.9, 28.4, 43.0; 2041 rows: 54.6, 61.3, 108; 3000 rows of 151000 with 8:
// 248, 225, 302.)
template <bool Bf16>
void launch_rows(const LogprobParams& p, hipStream_t stream) {
    const bool four_waves = p.vocab <= 16384 || (p.rows > 256 && p.vocab <= 65536);
    // (The threads of a launch stay below 2^32.)
    constexpr int64_t kMostRows = 1 << 22;
    for (int64_t first = 0; first < p.rows; first += kMostRows) {
        LogprobParams q = p;
        q.rows = std::min(p.rows - first, kMostRows);
        q.logits = static_cast<const uint8_t*>(p.logits) + first * p.stride * (Bf16 ? 2 : 4);
        q.tokens += first, q.logprob += first, q.entropy += first;
        if (p.top > 0) q.top_logprobs += first * p.top, q.top_tokens += first * p.top;
        const dim3 grid((unsigned)q.rows);
        if (four_waves)
            hipLaunchKernelGGL((logprobs_kernel<Bf16, 256>), grid, dim3(256), 0, stream, q);
        else
            hipLaunchKernelGGL((logprobs_kernel<Bf16, 512>), grid, dim3(512), 0, stream, q);
    }
}

}  // namespace

hipError_t launch_logprobs(const LogprobParams& p, hipStream_t stream) {
    if (p.bf16)
        launch_rows<true>(p, stream);
    else
        launch_rows<false>(p, stream);
    return hipGetLastError();
}

}  // namespace rq
