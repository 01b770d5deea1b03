// Verification of drafted tokens.  Row r of a request holds the distribution p_r
// of the token behind token t_r; all rows but the last have a draft t_{r+1},
// drawn from q_r.  With given random numbers u_r the draft is taken iff
// u_r q_r(t_{r+1}) < p_r(t_{r+1}); the first row whose draft is not, or the last
// row, is the final one.  Its token is drawn from the weights
// w = max(p - q, 0) (p in the last row) with the last row's u: the lowest token
// with w > 0 whose cumulative sum exceeds u times the whole.
//
// One launch: a workgroup finds a request's final row, sums some chunks of its weights
// and counts itself; the last of a request's workgroups finds the chunk and then,
// reading it once more, the token in it. (A launch of its own for the draw, a wave per
// request: 14.1 us for one request of 49152 tokens, 50.9 for 64 of 151000.) Bytes
// bound many requests, the chain of dependent loads a few: query starts, tokens, their
// probabilities, the numbers they are judged by, the request's last number, the row, the
// sums, the chunk. (Both kinds of numbers need the query starts alone, but are waited for in this order.)
//
// Sums are FP64: in FP32 their rounding, some 10^-7 of the whole, would move one
// border in thirty among 150000 tokens past a given u; in FP64 none.
#include <algorithm>

#include "rq_device.h"
#include "rq_plan.h"
#include "rq_reduced.h"

namespace rq {

namespace {

constexpr int kVerifyThreads = 256;

// What is no probability counts as 0.
__device__ __forceinline__ double probability(float p) { return p > 0.f && p < __builtin_inff() ? (double)p : 0.0; }

template <bool Bf16>
__device__ __forceinline__ float entry_of(const void* row, int64_t i) {
    return Bf16 ? bf16_f32(static_cast<const uint16_t*>(row)[i]) : static_cast<const float*>(row)[i];
}
template <bool Bf16>
__device__ __forceinline__ double probability_at(const void* row, int64_t i) { return probability(entry_of<Bf16>(row, i)); }

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

// Rows begin at any element.
typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef U32x4 U32x4At4 __attribute__((aligned(4)));
typedef U32x4 U32x4At2 __attribute__((aligned(2)));

// Entries of a row per 16-byte load, of a chunk's loads per thread: entry
// (256 k + thread) kEach + e of a chunk is load k's e.
template <bool Bf16>
constexpr int kEach = Bf16 ? 8 : 4;

template <bool Bf16>
__device__ __forceinline__ void load_entries(float (&x)[kEach<Bf16>], const void* row, int64_t at, int64_t vocab) {
    if (at + kEach<Bf16> <= vocab) {
        if constexpr (Bf16) {
            const U32x4 raw = *reinterpret_cast<const U32x4At2*>(static_cast<const uint16_t*>(row) + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[2 * e] = __uint_as_float(raw[e] << 16);
                x[2 * e + 1] = __uint_as_float(raw[e] & 0xffff0000u);
            }
        } else {
            const U32x4 raw = *reinterpret_cast<const U32x4At4*>(static_cast<const float*>(row) + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(raw[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < kEach<Bf16>; ++e) x[e] = at + e < vocab ? entry_of<Bf16>(row, at + e) : 0.f;
}

// This thread's weights of a chunk of a final row.
template <bool Bf16, int Loads>
__device__ __forceinline__ void chunk_weights(double (&w)[Loads][kEach<Bf16>], const VerifyParams& p, const VerifyRequest& r,
                                              int64_t chunk) {
    constexpr int E = kEach<Bf16>;
    const bool refused = r.end < r.stop - 1;
    const void* target = row_of<Bf16>(p.target, p.target_stride, r.end);
    const int64_t begin = chunk * (kVerifyThreads * E * Loads) + (int64_t)threadIdx.x * E;
    float of_target[Loads][E], of_draft[Loads][E];
#pragma unroll
    for (int k = 0; k < Loads; ++k) load_entries<Bf16>(of_target[k], target, begin + k * (kVerifyThreads * E), p.vocab);
    if (refused && p.draft != nullptr) {
        const void* draft = row_of<Bf16>(p.draft, p.draft_stride, r.end);
#pragma unroll
        for (int k = 0; k < Loads; ++k) load_entries<Bf16>(of_draft[k], draft, begin + k * (kVerifyThreads * E), p.vocab);
#pragma unroll
        for (int k = 0; k < Loads; ++k)
#pragma unroll
            for (int e = 0; e < E; ++e) w[k][e] = fmax(probability(of_target[k][e]) - probability(of_draft[k][e]), 0.0);
        return;
    }
    const int64_t without = refused ? p.tokens[r.end + 1] : -1;  // a refused draft that was certain
#pragma unroll
    for (int k = 0; k < Loads; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e)
            w[k][e] = begin + k * (kVerifyThreads * E) + e == without ? 0.0 : probability(of_target[k][e]);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
// Sum over the lanes up to this one.
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double below = __shfl_up(v, d);
        if (lane >= d) v += below;
    }
    return v;
}

// The first chunk whose running sum exceeds `limit` and whose own is above 0, else
// the last one above 0, else -1, and the running sum before it. For every wave by itself.
struct FoundChunk {
    int64_t chunk;
    double before, limit;  // limit: share x the sum of all
};
__device__ __forceinline__ FoundChunk find_chunk(const double* sums, int64_t chunks, double share) {
    const int lane = threadIdx.x & 63;
    auto sum_at = [&](int64_t c) {
        return c < chunks ? __longlong_as_double((long long)__hip_atomic_load(reinterpret_cast<const uint64_t*>(sums) + c, __ATOMIC_RELAXED,
                                                                              __HIP_MEMORY_SCOPE_AGENT)) : 0.0;
    };
    double whole = 0.0;
    const double first = sum_at(lane);  // (most rows have few chunks)
    for (int64_t base = 0; base < chunks; base += 64) whole += base == 0 ? first : sum_at(base + lane);
    const double limit = share * wave_sum(whole);
    FoundChunk found{-1, 0.0, limit};
    double before = 0.0;
    for (int64_t base = 0; base < chunks; base += 64) {
        const double own = base == 0 ? first : sum_at(base + lane), running = before + wave_scan(own);
        const uint64_t any = __ballot(own > 0.0), above = __ballot(own > 0.0 && running > limit);
        if (any != 0) {
            const int at = above != 0 ? __builtin_ctzll(above) : 63 - __builtin_clzll(any);
            found = FoundChunk{base + at, __shfl(running - own, at), limit};
            if (above != 0) break;
        }
        before = __shfl(running, 63);
    }
    return found;
}

// One workgroup per `p.each` (at most kMostChunks) chunks of a request's final row.
constexpr int kMostChunks = 8;
template <bool Bf16, int Loads>
__global__ __launch_bounds__(kVerifyThreads) void verify_kernel(const VerifyParams p) {
    constexpr int E = kEach<Bf16>, kWaves = kVerifyThreads / 64;
    __shared__ double sums_of[kMostChunks][kWaves];
    __shared__ int places[kWaves][2];
    __shared__ int last_flag;
    const int groups = (int)((p.chunks + p.each - 1) / p.each);  // workgroups of a request
    const int64_t request = blockIdx.x / groups, part = blockIdx.x % groups;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    uint64_t seen = 0;
    if (p.chunks > 1 && tid == 0) seen = peek_arrivals(p.arrivals + request * kVerifyArrivalStride);
    const VerifyRequest r = verify_request<Bf16>(p, request);
    if (part == 0) {
        // Rows outside of every request have no token.
        if (request == 0)
            for (int64_t row = tid; row < r.first; row += kVerifyThreads) p.out_tokens[row] = -1;
        if (request == p.requests - 1)
            for (int64_t row = r.stop + tid; row < p.rows; row += kVerifyThreads) p.out_tokens[row] = -1;
        for (int64_t row = r.first + tid; row < r.stop; row += kVerifyThreads)
            if (row != r.end) p.out_tokens[row] = row < r.end ? p.tokens[row + 1] : -1;
        if (tid == 0) p.accepted[request] = r.first == r.stop ? 0 : (int32_t)(r.end - r.first);
    }
    if (r.first == r.stop) return;
    double w[Loads][E], of_wave[Loads];
    FoundChunk found{0, 0.0, 0.0};
    const double share = (double)p.uniforms[r.stop - 1];
    double* const sums = p.sums + request * p.chunks;
    if (p.chunks > 1) {
        const int64_t chunk0 = part * p.each;
        const int count = (int)min((int64_t)p.each, p.chunks - chunk0);
        double sum[kMostChunks];
#pragma unroll
        for (int c = 0; c < kMostChunks; ++c) {
            if (c >= count) break;
            chunk_weights<Bf16, Loads>(w, p, r, chunk0 + c);
            sum[c] = 0.0;
#pragma unroll
            for (int k = 0; k < Loads; ++k)
#pragma unroll
                for (int e = 0; e < E; ++e) sum[c] += w[k][e];
        }
#pragma unroll
        for (int c = 0; c < kMostChunks; ++c) {
            if (c >= count) break;
            sum[c] = wave_sum(sum[c]);
            if (lane == 0) sums_of[c][wave] = sum[c];
        }
        if (tid == 0) tag_arrivals(p.arrivals + request * kVerifyArrivalStride, p.call_tag, seen);
        lds_barrier();
        if (tid < count) {
            double of_chunk = sums_of[tid][0];
#pragma unroll
            for (int v = 1; v < kWaves; ++v) of_chunk += sums_of[tid][v];
            __hip_atomic_store(reinterpret_cast<uint64_t*>(sums) + chunk0 + tid, (uint64_t)__double_as_longlong(of_chunk),
                               __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (!arrive_last_tagged(p.arrivals + request * kVerifyArrivalStride, groups, &last_flag)) return;
        found = find_chunk(sums, p.chunks, share);
        if (found.chunk < 0) {
            if (tid == 0) p.out_tokens[r.end] = -1;
            return;
        }
    }
    // The token in its chunk: running sums over load, wave, lane and entry.
    chunk_weights<Bf16, Loads>(w, p, r, found.chunk);
    double running[Loads];
#pragma unroll
    for (int k = 0; k < Loads; ++k) {
        double own = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) own += w[k][e];
        running[k] = wave_scan(own);
        of_wave[k] = running[k] - own;
        if (lane == 63) sums_of[k][wave] = running[k];
    }
    lds_barrier();
    double before = found.before, limit = found.limit;
    if (p.chunks == 1) {
        double whole = 0.0;
#pragma unroll
        for (int k = 0; k < Loads; ++k)
#pragma unroll
            for (int v = 0; v < kWaves; ++v) whole += sums_of[k][v];
        limit = share * whole;
    }
    constexpr int kNone = 0x7fffffff;
    int first = kNone, last = -1;  // of this thread: the first entry above the limit, the last above 0
#pragma unroll
    for (int k = 0; k < Loads; ++k) {
        double at = before + of_wave[k];
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            if (v < wave) at += sums_of[k][v];
            before += sums_of[k][v];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            at += w[k][e];
            const int place = (kVerifyThreads * k + tid) * E + e;
            if (w[k][e] > 0.0) {
                last = place;
                if (first == kNone && at > limit) first = place;
            }
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        first = min(first, __shfl_xor(first, d));
        last = max(last, __shfl_xor(last, d));
    }
    if (lane == 0) places[wave][0] = first, places[wave][1] = last;
    lds_barrier();
    if (tid == 0) {
#pragma unroll
        for (int v = 1; v < kWaves; ++v) first = min(first, places[v][0]), last = max(last, places[v][1]);
        const int place = first != kNone ? first : last;
        p.out_tokens[r.end] = place < 0 ? -1 : found.chunk * (kVerifyThreads * E * Loads) + place;
    }
}

// Loads per thread of a chunk: few where few requests leave compute units idle, at
// most as many as leave a row's chunks countable.
int loads_of(int64_t requests, int64_t vocab, bool bf16) {
    const int64_t least = kVerifyThreads * (bf16 ? 8 : 4);
    return requests * ((vocab + least - 1) / least) <= 1024 ? 1 : 4;
}

// Workgroups of a request: 1024 over all requests, but at least 8 (or one a chunk) and at most 64, as
// each finds the final row for itself and all count in one word; an eighth of the chunks
// where there are more than 512, as a workgroup takes at most kMostChunks. (One workgroup per
// chunk, the words of eight requests in a cache line: 64 requests of 151000 tokens 47.2 us
// and 18.1, 4 of them 21.1 and 9.6. At most 16, a line for each word: 18.5 and 13.1; 32: 18.2 and 10.8;
// 64, words side by side: 18.5 and 12.4.)
template <bool Bf16>
void launch(const VerifyParams& given, hipStream_t stream) {
    VerifyParams p = given;
    const int64_t most = std::min<int64_t>(std::max<int64_t>(1024 / p.requests, 8), 64);
    p.each = (int)std::min<int64_t>((p.chunks + most - 1) / most, kMostChunks);
    const dim3 grid((unsigned)(p.requests * ((p.chunks + p.each - 1) / p.each))), threads(kVerifyThreads);
    if (loads_of(p.requests, p.vocab, Bf16) == 1)
        hipLaunchKernelGGL((verify_kernel<Bf16, 1>), grid, threads, 0, stream, p);
    else
        hipLaunchKernelGGL((verify_kernel<Bf16, 4>), grid, threads, 0, stream, p);
}

}  // namespace

int64_t verify_chunks(int64_t requests, int64_t vocab, bool bf16) {
    const int64_t chunk = (int64_t)kVerifyThreads * (bf16 ? 8 : 4) * loads_of(requests, vocab, bf16);
    return (vocab + chunk - 1) / chunk;
}

hipError_t launch_verify(const VerifyParams& p, hipStream_t stream) {
    if (p.bf16)
        launch<true>(p, stream);
    else
        launch<false>(p, stream);
    return hipGetLastError();
}

}  // namespace rq
