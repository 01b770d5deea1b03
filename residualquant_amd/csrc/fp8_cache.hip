// Paged cache held in 8 bits: OCP E4M3 codes [2, blocks, kv_heads, PT, D] and
// one FP32 scale per (plane, block, head); a value is code * scale.
//
// quantize_fp8_kernel writes a call's new tokens, attention_fp8_kernel reads
// the cache: the 8-bit member beside the packed (2 + 4 bit) and the BF16 pages.
#include "rq_device.h"
#include "rq_plan.h"
#include "rq_reduced.h"

namespace rq {

namespace {

typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t U32x2 __attribute__((ext_vector_type(2)));
typedef U32x4 U32x4At8 __attribute__((aligned(8)));  // 16 bytes on an 8-byte boundary

// ------------------------------------------------------------------ write
//
// One wave per (page that the call writes, head, plane): the page's new
// values stay in registers between the maximum and the conversion, so each is
// read once.  Request b's pages take the slots from floor(first row / PT) + 2 b
// (n rows touch at most n / PT + 2 pages), so a wave finds its request by
// counting.

// The request of slot `slot` (the last whose first slot is at or below it).
__device__ __forceinline__ int write_request(const int32_t* qsl, int requests, int page_shift, int slot) {
    const int lane = threadIdx.x & 63;
    int count = 0;
    for (int b = 1 + lane; b < requests; b += 64) count += (int64_t)(qsl[b] >> page_shift) + 2 * (int64_t)b <= slot ? 1 : 0;
#pragma unroll
    for (int d = 32; d; d >>= 1) count += __shfl_xor(count, d);
    return __builtin_amdgcn_readfirstlane(count);
}

// The least power of two s >= 2^-126 with largest <= 448 s.  largest = m 2^e,
// 1 <= m < 2, and 448 = 1.75 * 2^8: s is 2^(e - 8), twice that where m > 1.75.
__device__ __forceinline__ float needed_scale(float largest) {
    const uint32_t u = __float_as_uint(largest);
    int exponent = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    if (exponent < 1) exponent = 1;  // 2^-126
    return __uint_as_float((uint32_t)exponent << 23);
}

// Four E4M3 codes (ties to even) of values within +-448; what is not finite becomes NaN.
__device__ __forceinline__ uint32_t fp8x4_rn(float a, float b, float c, float d) {
    auto nan_unless_finite = [](float x) { return fabsf(x) < __builtin_inff() ? x : __builtin_nanf(""); };
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(nan_unless_finite(a), nan_unless_finite(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(nan_unless_finite(c), nan_unless_finite(d), low, true);
}

__device__ __forceinline__ bool power_of_two(float x) { return (__float_as_uint(x) & 0x7fffffu) == 0; }

template <int D, int PT>
__global__ __launch_bounds__(256) void quantize_fp8_kernel(const Fp8WriteParams p) {
    constexpr int kRow = D / 8;                      // chunks of 8 values per row
    constexpr int kChunks = (PT * kRow + 63) / 64;   // per lane
    constexpr int kShift = PT == 16 ? 4 : 5;
    const int lane = threadIdx.x & 63;
    const int head = (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int plane = blockIdx.z;
    if (head >= p.kv_heads) return;
    const int request = write_request(p.query_start_loc, (int)p.requests, kShift, (int)blockIdx.x);
    const int first = p.query_start_loc[request];
    const int n = p.query_start_loc[request + 1] - first;
    const int64_t seq = p.seq_lens[request];
    const int64_t history = seq > n ? seq - n : 0;
    // The page: the slot's number among the request's, the rows from `begin` on at `slot`.
    const int64_t number = (int64_t)blockIdx.x - ((int64_t)(first >> kShift) + 2 * (int64_t)request);
    const int64_t page = (history >> kShift) + number;
    const int64_t begin = number == 0 ? 0 : (page << kShift) - history;
    if (n <= 0 || first < 0 || first + begin >= p.rows || number < 0 || begin >= n || page >= p.max_pages) return;
    const int slot = (int)((history + begin) & (PT - 1));
    const int rows = (int)min(min((int64_t)(PT - slot), n - begin), p.rows - first - begin);
    const int64_t block = p.block_table[(int64_t)request * p.block_table_stride + page];
    if (block < 0 || block >= p.num_blocks) return;
    const int64_t index = ((int64_t)plane * p.num_blocks + block) * p.kv_heads + head;
    uint8_t* const codes = p.cache + index * (PT * D);
    const float before = p.scales[index];
    const int64_t stride = plane == 0 ? p.key_stride : p.value_stride;
    const uint16_t* in = (plane == 0 ? p.key : p.value) + (first + begin) * stride + (int64_t)head * D;

    U32x4 values[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int chunk = 64 * c + lane, r = chunk / kRow;
        values[c] = U32x4{0u, 0u, 0u, 0u};
        if (r < rows) values[c] = *reinterpret_cast<const U32x4At8*>(in + r * stride + 8 * (chunk - r * kRow));
    }
    float largest = 0.f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = __uint_as_float(values[c][e] << 16), b = __uint_as_float(values[c][e] & 0xffff0000u);
            largest = fmaxf(largest, fabsf(a) < __builtin_inff() ? fabsf(a) : 0.f);
            largest = fmaxf(largest, fabsf(b) < __builtin_inff() ? fabsf(b) : 0.f);
        }
#pragma unroll
    for (int d = 32; d; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
    const float need = needed_scale(largest);
    const float scale = slot > 0 && before >= need ? before : need;

    if (slot > 0 && scale > before) {
        const float shrink = before / scale;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int chunk = 64 * c + lane;
            if (chunk >= slot * kRow) continue;
            U32x2* place = reinterpret_cast<U32x2*>(codes) + chunk;
            U32x2 word = *place;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(word[w], false), high = __builtin_amdgcn_cvt_pk_f32_fp8(word[w], true);
                word[w] = fp8x4_rn(low[0] * shrink, low[1] * shrink, high[0] * shrink, high[1] * shrink);
            }
            *place = word;
        }
    }
    // A division by a power of two is a product (a scale that the caller made may be any number).
    const bool exact = power_of_two(scale);
    const float inverse = 1.0f / scale;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int chunk = 64 * c + lane;
        if (chunk >= rows * kRow) continue;
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[2 * e] = __uint_as_float(values[c][e] << 16);
            x[2 * e + 1] = __uint_as_float(values[c][e] & 0xffff0000u);
        }
        if (exact) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= inverse;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] /= scale;
        }
        reinterpret_cast<U32x2*>(codes)[slot * kRow + chunk] =
            U32x2{fp8x4_rn(x[0], x[1], x[2], x[3]), fp8x4_rn(x[4], x[5], x[6], x[7])};
    }
    if (lane == 0) p.scales[index] = scale;
}

// ------------------------------------------------------------------ attention
//
// Queries are laid out as columns: the n new rows of a request times the
// `group` query heads that share a K/V head, column c = row (c / group), head
// c % group.  A wave streams the tokens of one (request, K/V head) for NT tiles
// of 16 columns, 32 tokens per step:
//   S^T = K Q^T    2 x D / 32 v_mfma_f32_16x16x32_bf16 (16 tokens x 16 columns),
//   O^T += V^T P^T  one per tile of 16 channels and part of P.
// Lane l = (i = l % 16, g = l / 16).  S^T leaves lane (q, g) the scores of
// tokens 4 g + r of both 16-token units for column q: exactly the slots that a
// B operand of the second product takes from this lane if its k slot
// (g, 4 u + r) stands for token 16 u + 4 g + r, so P never leaves the lane.
// The A operand then needs, per lane, channel (row) i of tokens 16 u + 4 g + r:
// lane (i, g) loads 8 channels 8 i.. of those 8 tokens and transposes 4 x 4
// bytes by v_perm; tile e holds channels 8 i + e, so lane (q, g) ends with the
// 32 channels 32 g.. of column q.  E4M3 becomes BF16 exactly.  Neither K nor V
// passes LDS.
//
// A page's K scale multiplies its scores (FP32), its V scale the weights
// (FP32), which are then split into two BF16 parts (16 bits of the weight
// multiply V; one part alone would round each weight by up to 2^-8, as much
// again as the rounding of the output.  A third part, for all 24 bits, changes
// one output of 600 by a BF16 step and the mean error against float64 in none of
// its first five digits, and takes 59.0 us instead of 57.7 for eight requests of
// five rows over 55 heads, 120 instead of 103 for two chunks of 509 rows).  The
// running maximum of a column moves only when a score exceeds it by 2^8, so most
// steps neither exchange lanes nor rescale; weights are then at most 2^8.
//
// Sums are not divided by the weights' sum before the end, so values near the
// top of BF16 would pass FP32 although their average does not.  From the first
// page scale above 2^72 or new value of 2^80 on, a wave counts O in units of
// 2^40: 2^30 tokens of any size then stay in range, and what the units lose is
// far below the rounding of such values.  The sign of a part's sum of weights
// says in which unit its O is.  All of it lies on paths that are rare already
// (tokens that do not count, values that are not finite): no time.  (A second
// pass after an overflow: 11.4 us of 10.5 for one request of 2048 tokens, and 152
// bytes of spilled registers where there are many columns.)

typedef __bf16 Bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 Bf16x2 __attribute__((ext_vector_type(2)));
typedef float F32x4 __attribute__((ext_vector_type(4)));

constexpr int kStreamThreads = 256;
constexpr float kLowest = -3.402823466e+38f;
constexpr float kMaxSlack = 8.0f;  // log2 units
constexpr float kHugeUnit = 0x1p40f, kHugeScale = 0x1p72f, kHugeValue = 0x1p80f;

__device__ __forceinline__ F32x4 mfma(U32x4 a, U32x4 b, F32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Bf16x8, a), __builtin_bit_cast(Bf16x8, b), c, 0, 0, 0);
}

// Two E4M3 codes (low or high half word of x) as two BF16, exactly.
template <bool High>
__device__ __forceinline__ uint32_t bf16x2_of_fp8(uint32_t x) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, High));
}

// t[c] = byte c of x[0..3] (x[0] lowest).
__device__ __forceinline__ void transpose_bytes(const uint32_t (&x)[4], uint32_t (&t)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400);  // x0.0 x1.0 x0.1 x1.1
    const uint32_t b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400);
    const uint32_t c = __builtin_amdgcn_perm(x[1], x[0], 0x07030602);  // x0.2 x1.2 x0.3 x1.3
    const uint32_t d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602);
    t[0] = __builtin_amdgcn_perm(b, a, 0x05040100);
    t[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
    t[2] = __builtin_amdgcn_perm(d, c, 0x05040100);
    t[3] = __builtin_amdgcn_perm(d, c, 0x07060302);
}

// Values that the products leave out and that are added apart: of kHugeValue and more, infinities, NaN.
__device__ __forceinline__ bool odd_bf16x2(uint32_t x) {
    return (x & 0x7f80u) >= 0x6780u || (x & 0x7f800000u) >= 0x67800000u;
}
__device__ __forceinline__ uint32_t without_odd(uint32_t x) {
    if ((x & 0x7f80u) >= 0x6780u) x &= 0xffff0000u;
    if ((x & 0x7f800000u) >= 0x67800000u) x &= 0x0000ffffu;
    return x;
}

// One request's new rows (as columns) and history.
struct Fp8Request {
    int first, rows, history;
};

__device__ __forceinline__ Fp8Request fp8_request(const Fp8AttentionParams& p, int request) {
    Fp8Request r;
    r.first = p.query_start_loc[request];
    const int n = p.query_start_loc[request + 1] - r.first;
    // Rows past the query tensor are not read or written.
    r.rows = r.first < 0 || r.first >= p.rows ? 0 : (int)min((int64_t)max(n, 0), p.rows - r.first);
    const int seq = p.seq_lens[request];
    // Tokens past the page table are never read.
    r.history = p.num_blocks > 0 ? (int)min((int64_t)(seq > n ? (int64_t)seq - n : 0), p.max_pages * p.page_tokens) : 0;
    return r;
}

// Steps (of 32 tokens) of a request: its history, then its new rows.
__device__ __forceinline__ int fp8_steps(int tokens) { return (tokens + 31) / 32; }

// The item of a workgroup: PlanItem's rows are columns, its length steps.
template <int Tile>
__device__ __forceinline__ PlanItem fp8_item(const Fp8AttentionParams& p, int key) {
    const int group = p.heads / p.kv_heads, requests = (int)p.requests;
    const int lane = threadIdx.x & 63;
    if (p.items > 0) {
        const Fp8Request q = fp8_request(p, lane < requests ? lane : requests - 1);
        const int columns = lane < requests ? q.rows * group : 0;
        const PlanEntry own{(columns + Tile - 1) / Tile, fp8_steps(q.history) + fp8_steps(q.rows), q.first, q.history, columns};
        const PlanSizes sizes = fp8_sizes(p);
        PlanItem item = plan_find(requests, key, sizes, own);
        // (Query starts that do not ascend could ask for more entries than the workspace has.)
        if (item.splits > 1 && (item.entry < 0 || item.entry + (int64_t)item.rows * item.splits > p.entries)) item.request = -1;
        return item;
    }
    // More requests than a wave has lanes: tile i of request b has slot
    // floor(first column of b / Tile) + b + i, each slot `splits` workgroups.
    const int slot = key / p.splits;
    int count = 0;
    for (int b = 1 + lane; b < requests; b += 64)
        count += (int64_t)p.query_start_loc[b] * group / Tile + b <= slot ? 1 : 0;
#pragma unroll
    for (int d = 32; d; d >>= 1) count += __shfl_xor(count, d);
    const Fp8Request q = fp8_request(p, count);
    const int index = slot - (int)((int64_t)q.first * group / Tile + count);
    const int columns = q.rows * group;
    if (index < 0 || index * Tile >= columns) return PlanItem{-1, 0, 0, 1, 0, 0, 0, 0, 0, 0, 0};
    return PlanItem{count, index, key % p.splits, p.splits, fp8_steps(q.history) + fp8_steps(q.rows), q.first, q.history,
                    columns, 0, q.first * group * p.splits, 0};
}

// Codes of one step: 16 tokens' K rows and this lane's 8 tokens of V, for both units.
template <int D>
struct Fp8Step {
    U32x4 k[2][D == 128 ? 2 : 1];
    U32x2 k_rest[2];  // D = 96
    U32x2 v[2][4];
    float key_scale[2], value_scale[2];
    int valid[2];  // tokens of the unit inside the history
};

// The columns' statistics and sums of a wave.
template <int NT, int Channels>
struct Fp8Columns {
    F32x4 out[NT][Channels];  // [tile][e]
    float high[NT];  // the maximum that weights refer to (log2 units)
    float sum[NT];   // of this lane's tokens
    float unit;      // by which O is multiplied (the same for the whole wave): 1 or 1 / kHugeUnit

    __device__ __forceinline__ void clear() {
        unit = 1.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            high[t] = kLowest;
            sum[t] = 0.f;
#pragma unroll
            for (int e = 0; e < Channels; ++e) out[t][e] = F32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void make_room() {
        if (unit != 1.0f) return;
        unit = 1.0f / kHugeUnit;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < Channels; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) out[t][e][r] *= 1.0f / kHugeUnit;
    }
    // A part's sum as it is handed on.
    __device__ __forceinline__ float marked_sum(int t) const { return unit == 1.0f ? sum[t] : -sum[t]; }
};

// Of the parts of a column, `marks`: their sums' bits, or-ed (without branches, beside loads in flight).
// What a part's O counts in the join's unit, and that unit over the sum.
__device__ __forceinline__ float part_unit(uint32_t marks, float sum) {
    return (int)(marks & ~__float_as_uint(sum)) < 0 ? 1.0f / kHugeUnit : 1.0f;
}
__device__ __forceinline__ float join_scale(uint32_t marks, float sum) { return ((int)marks < 0 ? kHugeUnit : 1.0f) / sum; }

// a * b, rounded also where a sum follows.  (A score less the maximum by one fma would be its product's
// rounding away from 0 at the maximum itself: from scores of 2^31 on that is a weight of 2^128, or none.
// No time in any kernel.)
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// A page's K scale with the softmax scale: positive also where the product is too small for FP32 (0 would
// make NaN of the -inf of masked scores).
__device__ __forceinline__ float factor_of_scores(float scale, float to_log2) { return fmaxf(scale * to_log2, 0x1p-149f); }

// Weights of U units of 16 tokens: of the products dot (masked: -inf) with their
// K scales (positive, softmax scale and log2(e) included), as two BF16 parts of
// weight x V scale.  Channels: the product's tiles of 16.
template <int NT, int Channels, int U>
__device__ __forceinline__ void fp8_softmax(Fp8Columns<NT, Channels>& columns, const F32x4 (&dot)[NT][U],
                                            const float (&key_scale)[U], const float (&value_scale)[U],
                                            float (&weight)[NT][U][4], U32x4 (&upper)[NT][U / 2], U32x4 (&lower)[NT][U / 2]) {
    float top[NT];
    bool above = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        top[t] = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < U; ++u)
            top[t] = fmaxf(top[t], fmaxf(fmaxf(dot[t][u][0], dot[t][u][1]), fmaxf(dot[t][u][2], dot[t][u][3])) * key_scale[u]);
        above = above || top[t] > columns.high[t] + kMaxSlack;
    }
    if (__any(above)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            top[t] = fmaxf(top[t], __shfl_xor(top[t], 16));
            top[t] = fmaxf(top[t], __shfl_xor(top[t], 32));
            const float next = fmaxf(columns.high[t], top[t]);
            const float keep = next == columns.high[t] ? 1.0f : __builtin_amdgcn_exp2f(columns.high[t] - next);
            columns.high[t] = next;
            columns.sum[t] *= keep;
#pragma unroll
            for (int e = 0; e < Channels; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) columns.out[t][e][r] *= keep;
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        uint32_t up[2 * U], low[2 * U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                weight[t][u][r] = __builtin_amdgcn_exp2f(rounded_product(dot[t][u][r], key_scale[u]) - columns.high[t]);
                columns.sum[t] += weight[t][u][r];
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float a = weight[t][u][2 * h] * value_scale[u], b = weight[t][u][2 * h + 1] * value_scale[u];
                const uint32_t both = bf16x2_rn(a, b);
                up[2 * u + h] = both;
                low[2 * u + h] = bf16x2_rn(a - __uint_as_float(both << 16), b - __uint_as_float(both & 0xffff0000u));
            }
        }
#pragma unroll
        for (int s = 0; s < U / 2; ++s) {
            upper[t][s] = U32x4{up[4 * s], up[4 * s + 1], up[4 * s + 2], up[4 * s + 3]};
            lower[t][s] = U32x4{low[4 * s], low[4 * s + 1], low[4 * s + 2], low[4 * s + 3]};
        }
    }
}

// Joins the splits' parts of columns from..to - 1, in the splits' order.  Shared:
// they come from workgroups of the same launch, past the caches that are not coherent.
template <int D, int Threads, bool Shared, class OutputRow>
__device__ __forceinline__ void fp8_join(__amdgpu_buffer_rsrc_t handoff, int from, int to, int splits, OutputRow output_row) {
    constexpr int kEntry = D + 4;
    const int tid = threadIdx.x, channel = 8 * (tid & 15);
    if (channel >= D) return;
    for (int column = from + (tid >> 4); column < to; column += Threads / 16) {
        const uint32_t at = (uint32_t)(column * splits) * kEntry * 4;
        // Parts in groups of four whose loads are all in flight (past the last part that one again, with a weight
        // of 0), the first group together with the maxima of the others: one wait for up to four parts, and no
        // chain of rescaled sums for more. One pass with rescaling took 11.1 us against 9.8 for one request of
        // 2048 tokens; loads that wait part by part 118 us against 113 for a chunk of 512 rows.
        constexpr int kGroup = 4;
        float2 stats[kGroup];
        float4 low[kGroup], up[kGroup];
        const auto load2 = [&](uint32_t place) {
            if constexpr (Shared) return handoff_load2(handoff, place);
            const U32x2 v = __builtin_amdgcn_raw_buffer_load_b64(handoff, place, 0, 0);
            return make_float2(__uint_as_float(v[0]), __uint_as_float(v[1]));
        };
        const auto load4 = [&](uint32_t place) {
            if constexpr (Shared) return handoff_load4(handoff, place);
            const U32x4 v = __builtin_amdgcn_raw_buffer_load_b128(handoff, place, 0, 0);
            return make_float4(__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2]), __uint_as_float(v[3]));
        };
        const auto load = [&](int first) {
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
                const uint32_t part = at + (uint32_t)min(first + k, splits - 1) * kEntry * 4;
                stats[k] = load2(part);
                low[k] = load4(part + 16 + 4 * channel);
                up[k] = load4(part + 32 + 4 * channel);
            }
        };
        load(0);
        float high = kLowest;
        uint32_t marks = 0;
        for (int first = kGroup; first < splits; first += 8) {
            float2 others[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) others[k] = load2(at + (uint32_t)min(first + k, splits - 1) * kEntry * 4);
#pragma unroll
            for (int k = 0; k < 8; ++k) high = fmaxf(high, others[k].x), marks |= __float_as_uint(others[k].y);
        }
#pragma unroll
        for (int k = 0; k < kGroup; ++k) high = fmaxf(high, stats[k].x), marks |= __float_as_uint(stats[k].y);
        float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
        for (int first = 0;;) {
#pragma unroll
            for (int k = 0; k < kGroup; ++k) {
                float keep = first + k >= splits ? 0.0f : stats[k].x == high ? 1.0f : __builtin_amdgcn_exp2f(stats[k].x - high);
                sum += fabsf(stats[k].y) * keep;
                keep *= part_unit(marks, stats[k].y);
                o[0] += low[k].x * keep, o[1] += low[k].y * keep, o[2] += low[k].z * keep, o[3] += low[k].w * keep;
                o[4] += up[k].x * keep, o[5] += up[k].y * keep, o[6] += up[k].z * keep, o[7] += up[k].w * keep;
            }
            first += kGroup;
            if (first >= splits) break;
            load(first);
        }
        const float scale = join_scale(marks, sum);
        uint16_t* out = output_row(column) + channel;
        *reinterpret_cast<U32x2*>(out) = U32x2{bf16x2_rn(o[0] * scale, o[1] * scale), bf16x2_rn(o[2] * scale, o[3] * scale)};
        *reinterpret_cast<U32x2*>(out + 4) = U32x2{bf16x2_rn(o[4] * scale, o[5] * scale), bf16x2_rn(o[6] * scale, o[7] * scale)};
    }
}

// One workgroup per (item, K/V head): its four waves take every fourth step of
// the item's 16 NT columns.
template <int D, int NT>
__global__ __launch_bounds__(kStreamThreads) void attention_fp8_kernel(const Fp8AttentionParams p) {
    constexpr int kTile = 16 * NT, kWaves = kStreamThreads / 64;
    constexpr int kSteps = D / 32;
    constexpr int kEntry = D + 4;  // m, l, arrival word, O
    __shared__ __align__(16) float merged[kWaves][16][kEntry];
    __shared__ int last_flag;
    const int head = (int)(blockIdx.x % (unsigned)p.kv_heads);
    const PlanItem item = fp8_item<kTile>(p, (int)(blockIdx.x / (unsigned)p.kv_heads));
    const int request = __builtin_amdgcn_readfirstlane(item.request);
    if (request < 0) return;  // uniform over the workgroup, before any barrier
    const int group = p.heads / p.kv_heads;
    const int first = __builtin_amdgcn_readfirstlane(item.first), columns_in = __builtin_amdgcn_readfirstlane(item.rows);
    const int rows = columns_in / group;
    const int history = __builtin_amdgcn_readfirstlane(item.tokens);
    const int splits = __builtin_amdgcn_readfirstlane(item.splits), split = __builtin_amdgcn_readfirstlane(item.split);
    const int begin = split_begin(__builtin_amdgcn_readfirstlane(item.length), split, splits);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int item_column = __builtin_amdgcn_readfirstlane(item.index) * kTile;
    const int end = split_begin(__builtin_amdgcn_readfirstlane(item.length), split + 1, splits);
    const int history_steps = fp8_steps(history);

    // The item's arrival word lies in the two unused floats of its first entry.
    float* const entries = p.partials + ((int64_t)head * p.entries + __builtin_amdgcn_readfirstlane(item.entry)) * kEntry;
    uint64_t* const arrivals = reinterpret_cast<uint64_t*>(entries + (int64_t)item_column * splits * kEntry + 2);
    const uint64_t arrivals_seen = splits > 1 ? peek_arrivals(arrivals) : 0;

    // Queries: column q's channels of each k step (the K loads' order), and the
    // last new row that the column sees.
    U32x4 query[NT][kSteps];
    int seen[NT];
    auto k_channel = [&](int s) { return D == 128 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 24 * g + 8 * s; };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int column = item_column + 16 * t + i;
        seen[t] = column < columns_in ? column / group : -1;
        const int row = column < columns_in ? column / group : 0;
        const uint16_t* q = p.query + (int64_t)(first + row) * p.query_stride +
                            ((int64_t)head * group + (column < columns_in ? column % group : 0)) * D;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const U32x2 a = *reinterpret_cast<const U32x2*>(q + k_channel(s));
            const U32x2 b = *reinterpret_cast<const U32x2*>(q + k_channel(s) + 4);
            query[t][s] = column < columns_in ? U32x4{a[0], a[1], b[0], b[1]} : U32x4{0u, 0u, 0u, 0u};
        }
    }
    Fp8Columns<NT, 8> columns;  // tile e: channels 8 (4 g + r) + e
    columns.clear();
    const float to_log2 = p.softmax_scale * 1.44269504088896341f;

    // ---------------------------------------------------------------- history
    // Lane l holds the place, scales and valid tokens of unit l % 2 of the
    // wave's step l / 2 of a batch of 32.
    const int page_shift = p.page_tokens == 16 ? 4 : 5;
    const int64_t plane_bytes = ((p.num_blocks * p.kv_heads) << page_shift) * D;
    const int step0 = begin + wave;
    const int my_steps = max(0, (min(end, history_steps) - step0 + kWaves - 1) / kWaves);
    uint32_t place_low = 0, place_high = 0, unit_valid = 0;
    float unit_key_scale = 1.f, unit_value_scale = 1.f;
    auto look_up = [&](int batch) {
        const int step = step0 + (32 * batch + (lane >> 1)) * kWaves;
        const int token = 32 * step + 16 * (lane & 1);
        const int left = step < min(end, history_steps) ? history - token : 0;
        const int page = token >> page_shift;
        int64_t block = left > 0 ? p.block_table[(int64_t)request * p.block_table_stride + page] : -1;
        const bool held = block >= 0 && block < p.num_blocks;
        if (!held) block = 0;
        const int64_t index = block * p.kv_heads + head;
        const int64_t place = ((index << page_shift) + (token & (p.page_tokens - 1))) * D;
        place_low = (uint32_t)place;
        place_high = (uint32_t)((uint64_t)place >> 32);
        unit_valid = held ? (uint32_t)min(left, 16) : 0u;
        unit_key_scale = held ? factor_of_scores(p.scales[index], to_log2) : 1.f;
        unit_value_scale = held ? p.scales[index + p.num_blocks * p.kv_heads] : 1.f;
    };
    auto load = [&](Fp8Step<D>& x, int number) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int from = 2 * (number & 31) + u;
            const int64_t place = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane(place_high, from) << 32) |
                                            (uint32_t)__builtin_amdgcn_readlane(place_low, from));
            x.valid[u] = __builtin_amdgcn_readlane(unit_valid, from);
            x.key_scale[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(unit_key_scale), from));
            x.value_scale[u] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(unit_value_scale), from));
            const uint8_t* k = p.cache + place;
            const uint8_t* v = k + plane_bytes;
            if constexpr (D == 128) {
                x.k[u][0] = *reinterpret_cast<const U32x4*>(k + (i * D + 16 * g));
                x.k[u][1] = *reinterpret_cast<const U32x4*>(k + (i * D + 16 * g + 64));
            } else {
                const U32x2 a = *reinterpret_cast<const U32x2*>(k + (i * D + 24 * g));
                const U32x2 b = *reinterpret_cast<const U32x2*>(k + (i * D + 24 * g + 8));
                x.k[u][0] = U32x4{a[0], a[1], b[0], b[1]};
                x.k_rest[u] = *reinterpret_cast<const U32x2*>(k + (i * D + 24 * g + 16));
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x.v[u][r] = *reinterpret_cast<const U32x2*>(v + ((4 * g + r) * D + (8 * i < D ? 8 * i : 0)));
        }
    };
    auto compute = [&](const Fp8Step<D>& x) {
        F32x4 dot[NT][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int t = 0; t < NT; ++t) dot[t][u] = F32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < kSteps; ++m) {
                uint32_t a0, a1;
                if constexpr (D == 128) {
                    a0 = x.k[u][m >> 1][2 * (m & 1)], a1 = x.k[u][m >> 1][2 * (m & 1) + 1];
                } else {
                    a0 = m < 2 ? x.k[u][0][2 * (m & 1)] : x.k_rest[u][0];
                    a1 = m < 2 ? x.k[u][0][2 * (m & 1) + 1] : x.k_rest[u][1];
                }
                const U32x4 a = {bf16x2_of_fp8<false>(a0), bf16x2_of_fp8<true>(a0), bf16x2_of_fp8<false>(a1),
                                 bf16x2_of_fp8<true>(a1)};
#pragma unroll
                for (int t = 0; t < NT; ++t) dot[t][u] = mfma(a, query[t][m], dot[t][u]);
            }
        }
        // (Scalar instructions: positive floats compare as their bits.)
        const bool whole = min(x.valid[0], x.valid[1]) == 16;
        const bool huge = max(__float_as_uint(x.value_scale[0]), __float_as_uint(x.value_scale[1])) > __builtin_bit_cast(uint32_t, kHugeScale);
        if (!whole || huge) {
            if (huge) columns.make_room();
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        dot[t][u][r] = 4 * g + r < x.valid[u] ? dot[t][u][r] : -__builtin_inff();
        }
        float weight[NT][2][4];
        U32x4 upper[NT][1], lower[NT][1];
        const float value_scale[2] = {x.value_scale[0] * columns.unit, x.value_scale[1] * columns.unit};
        fp8_softmax<NT, 8, 2>(columns, dot, x.key_scale, value_scale, weight, upper, lower);
        uint32_t v[2][4][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int w = 0; w < 2; ++w) v[u][r][w] = x.v[u][r][w];
        // Slots past the history may hold NaN, which a weight of zero does not remove.
        if (!whole) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int w = 0; w < 2; ++w) v[u][r][w] = 4 * g + r < x.valid[u] ? v[u][r][w] : 0u;
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            uint32_t t0[4], t1[4];
            const uint32_t x0[4] = {v[0][0][w], v[0][1][w], v[0][2][w], v[0][3][w]};
            const uint32_t x1[4] = {v[1][0][w], v[1][1][w], v[1][2][w], v[1][3][w]};
            transpose_bytes(x0, t0);
            transpose_bytes(x1, t1);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const U32x4 a = {bf16x2_of_fp8<false>(t0[c]), bf16x2_of_fp8<true>(t0[c]), bf16x2_of_fp8<false>(t1[c]),
                                 bf16x2_of_fp8<true>(t1[c])};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    columns.out[t][4 * w + c] = mfma(a, upper[t][0], columns.out[t][4 * w + c]);
                    columns.out[t][4 * w + c] = mfma(a, lower[t][0], columns.out[t][4 * w + c]);
                }
            }
        }
    };
    // (Loads without a condition, past the last step of that step again: after a
    // load that one path leaves out, every wait would be for all loads in flight.)
    if (my_steps > 0) {
        Fp8Step<D> even, odd;
        look_up(0);
        load(even, 0);
        for (int n = 0; n < my_steps; n += 2) {
            load(odd, min(n + 1, my_steps - 1));
            compute(even);
            if (n + 1 >= my_steps) break;
            if (((n + 2) & 31) == 0) look_up((n + 2) >> 5);
            load(even, min(n + 2, my_steps - 1));
            compute(odd);
        }
    }

    // ---------------------------------------------------------------- new rows
    // (BF16 rows of this call, row j seen by the columns of rows j and later.)
    {
        const int most = min(rows - 1, (item_column + 16 * NT - 1) / group);  // the last row that any column sees
        int step = step0;
        if (step < history_steps) step += (history_steps - step + kWaves - 1) / kWaves * kWaves;
        for (; step < end; step += kWaves) {
            const int base = 32 * (step - history_steps);
            if (base > most) break;
            F32x4 dot[NT][2];
            U32x4 v[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int t = 0; t < NT; ++t) dot[t][u] = F32x4{0.f, 0.f, 0.f, 0.f};
                const uint16_t* k = p.key + (int64_t)(first + min(base + 16 * u + i, rows - 1)) * p.key_stride + (int64_t)head * D;
#pragma unroll
                for (int m = 0; m < kSteps; ++m) {
                    const U32x2 a = *reinterpret_cast<const U32x2*>(k + k_channel(m));
                    const U32x2 b = *reinterpret_cast<const U32x2*>(k + k_channel(m) + 4);
#pragma unroll
                    for (int t = 0; t < NT; ++t) dot[t][u] = mfma(U32x4{a[0], a[1], b[0], b[1]}, query[t][m], dot[t][u]);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int token = base + 16 * u + 4 * g + r;
#pragma unroll
                    for (int t = 0; t < NT; ++t) dot[t][u][r] = token <= seen[t] ? dot[t][u][r] : -__builtin_inff();
                    const uint16_t* row = p.value + (int64_t)(first + min(token, rows - 1)) * p.value_stride +
                                          (int64_t)head * D + (8 * i < D ? 8 * i : 0);
                    const U32x2 a = *reinterpret_cast<const U32x2*>(row), b = *reinterpret_cast<const U32x2*>(row + 4);
                    v[u][r] = U32x4{a[0], a[1], b[0], b[1]};
                }
            }
            float weight[NT][2][4];
            U32x4 upper[NT][1], lower[NT][1];
            const float key_scale[2] = {to_log2, to_log2}, value_scale[2] = {columns.unit, columns.unit};
            fp8_softmax<NT, 8, 2>(columns, dot, key_scale, value_scale, weight, upper, lower);
            // Infinities and NaN, which a weight of zero does not remove, and huge values are added apart.
            bool odd_values = false;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int w = 0; w < 4; ++w) odd_values |= odd_bf16x2(v[u][r][w]);
            const bool any_odd = __any(odd_values);
            if (any_odd) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int w = 0; w < 4; ++w) v[u][r][w] = without_odd(v[u][r][w]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t pick = e & 1 ? 0x07060302u : 0x05040100u;  // the upper or lower halves of two words
                const U32x4 a = {__builtin_amdgcn_perm(v[0][1][e >> 1], v[0][0][e >> 1], pick),
                                 __builtin_amdgcn_perm(v[0][3][e >> 1], v[0][2][e >> 1], pick),
                                 __builtin_amdgcn_perm(v[1][1][e >> 1], v[1][0][e >> 1], pick),
                                 __builtin_amdgcn_perm(v[1][3][e >> 1], v[1][2][e >> 1], pick)};
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    columns.out[t][e] = mfma(a, upper[t][0], columns.out[t][e]);
                    columns.out[t][e] = mfma(a, lower[t][0], columns.out[t][e]);
                }
            }
            if (any_odd) {
                columns.make_room();
                for (int j = 0; j < 32; ++j) {
                    const int token = base + j;
                    if (token >= rows) break;
                    const uint16_t* row = p.value + (int64_t)(first + token) * p.value_stride + (int64_t)head * D;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        // (selected without an index, so that the weights stay in registers)
                        float mine = 0.f;
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (16 * u + r == (j & 19)) mine = weight[t][u][r];
                        const float w = __shfl(mine, i + 16 * ((j >> 2) & 3));
                        if (token > seen[t]) continue;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const int channel = 32 * g + 8 * r + e;
                                if (channel >= D) continue;
                                const float x = bf16_f32(row[channel]);
                                if (!(fabsf(x) < kHugeValue)) columns.out[t][e][r] += w * (x * columns.unit);
                            }
                    }
                }
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        columns.sum[t] += __shfl_xor(columns.sum[t], 16);
        columns.sum[t] += __shfl_xor(columns.sum[t], 32);
    }

    // ---------------------------------------------------------------- finish
    const __amdgpu_buffer_rsrc_t handoff = handoff_resource(entries, (uint32_t)min((int64_t)columns_in * splits * kEntry * 4, (int64_t)0xfffffffc));
    auto output_row = [&](int column) {
        return p.output + (int64_t)(first + column / group) * p.output_stride + ((int64_t)head * group + column % group) * D;
    };
    // Eight channels of a column: the output, or this split's part of it.
    auto emit = [&](int column, int channel, const float (&o)[8], float high, float sum, uint32_t marks) {
        if (splits == 1) {
            const float scale = join_scale(marks, sum);
            uint16_t* out = output_row(column) + channel;
            *reinterpret_cast<U32x2*>(out) = U32x2{bf16x2_rn(o[0] * scale, o[1] * scale), bf16x2_rn(o[2] * scale, o[3] * scale)};
            *reinterpret_cast<U32x2*>(out + 4) = U32x2{bf16x2_rn(o[4] * scale, o[5] * scale), bf16x2_rn(o[6] * scale, o[7] * scale)};
            return;
        }
        const uint32_t at = (uint32_t)(column * splits + split) * kEntry * 4;
        handoff_store4(handoff, at + 16 + 4 * channel, o[0], o[1], o[2], o[3]);
        handoff_store4(handoff, at + 32 + 4 * channel, o[4], o[5], o[6], o[7]);
        if (channel == 0) {
            handoff_store(handoff, at, high);
            handoff_store(handoff, at + 4, (int)marks < 0 ? -sum : sum);
        }
    };
    if (splits > 1 && tid == 0) tag_arrivals(arrivals, p.call_tag, arrivals_seen);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int channel = 32 * g + 8 * r;
            if (channel >= D) continue;
            float* to = &merged[wave][i][channel];
            *reinterpret_cast<F32x4*>(to) = F32x4{columns.out[t][0][r], columns.out[t][1][r], columns.out[t][2][r], columns.out[t][3][r]};
            *reinterpret_cast<F32x4*>(to + 4) = F32x4{columns.out[t][4][r], columns.out[t][5][r], columns.out[t][6][r], columns.out[t][7][r]};
        }
        if (g == 0) {
            merged[wave][i][D] = columns.high[t];
            merged[wave][i][D + 1] = columns.marked_sum(t);
        }
        __syncthreads();
        const int local = tid >> 4, channel = 8 * (tid & 15), column = item_column + 16 * t + local;
        if (column < columns_in && channel < D) {
            float high = kLowest;
            uint32_t marks = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w)
                high = fmaxf(high, merged[w][local][D]), marks |= __float_as_uint(merged[w][local][D + 1]);
            float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float m = merged[w][local][D];
                float keep = m == high ? 1.0f : __builtin_amdgcn_exp2f(m - high);
                sum += fabsf(merged[w][local][D + 1]) * keep;
                keep *= part_unit(marks, merged[w][local][D + 1]);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += merged[w][local][channel + e] * keep;
            }
            emit(column, channel, o, high, sum, marks);
        }
    }
    if (splits == 1 || !arrive_last_tagged(arrivals, splits, &last_flag)) return;
    // The last split to finish joins.
    fp8_join<D, kStreamThreads, true>(handoff, item_column, min(item_column + kTile, columns_in), splits, output_row);
}

// ------------------------------------------------------------------ many columns
//
// The same products for requests of many columns: eight waves of 32 columns
// share tiles of 64 tokens, which they convert to BF16 once, into LDS:
// K as it is read ([token][channel]), V transposed ([channel][token], the tokens
// in the order in which the second product's k slots stand for them).  Rows of
// 256 and 128 bytes; the 16-byte chunks of a row are permuted by its number so
// that the 16 rows an operand read touches lie in different banks.  A tile's
// global loads are issued a tile ahead and converted into the other buffer
// after the products of the present one: one barrier per tile.
//
// One request of 8192 tokens + 1024 new rows, 16 heads of 128: 147 us, 3.8 us per
// tile and compute unit, of which the matrix units work 1.6 (a third of it for the
// weights' lower parts); the rest is the vector instructions of the weights and
// conversions, about as long, and waits for LDS.  Two waves per SIMD hide
// little of one another; four (16 columns each) spill registers (224 us), one
// of 64 columns took 276, and the weights of one step beside the products of
// the other in one wave 154.

constexpr int kWideTokens = 64, kWideThreads = 512, kWideColumns = 32;  // columns of a wave
constexpr int kWideTile = kWideColumns * kWideThreads / 64;

// Distinct for channels c..c + 7 (an operand read) and for every fourth (the transposing writes).
__device__ __forceinline__ int v_swizzle(int channel) { return (channel ^ (channel >> 2)) & 7; }

constexpr int kHugeFlag = 32;  // of a unit whose page has a V scale above kHugeScale

template <int D>
struct WideTile {
    U32x4 k[kWideTokens][16];  // [token][chunk of 8 channels, chunk ^ (token % 16)]
    U32x4 v[D][8];             // [channel][chunk of 8 tokens, chunk ^ v_swizzle(channel)]
    float key_scale[4], value_scale[4];  // of the tile's units of 16 tokens
    int valid[4];              // tokens of the unit that count (0 to 16), and kHugeFlag
    int odd;                   // the number of the last tile of new rows with odd_bf16x2 among its values
};

template <int D>
__global__ __launch_bounds__(kWideThreads) void attention_fp8_wide_kernel(const Fp8AttentionParams p) {
    constexpr int NT = kWideColumns / 16, kTile = kWideTile, kSteps = D / 32, kOut = D / 16, kEntry = D + 4;
    constexpr int kChunks = D / 16;               // 16-byte chunks of a row of codes
    __shared__ WideTile<D> tiles[2];
    const int head = (int)(blockIdx.x % (unsigned)p.kv_heads);
    const PlanItem item = fp8_item<kTile>(p, (int)(blockIdx.x / (unsigned)p.kv_heads));
    const int request = __builtin_amdgcn_readfirstlane(item.request);
    if (request < 0) return;  // uniform over the workgroup, before any barrier
    const int group = p.heads / p.kv_heads;
    const int first = __builtin_amdgcn_readfirstlane(item.first), columns_in = __builtin_amdgcn_readfirstlane(item.rows);
    const int rows = columns_in / group;
    const int history = __builtin_amdgcn_readfirstlane(item.tokens);
    const int splits = __builtin_amdgcn_readfirstlane(item.splits), split = __builtin_amdgcn_readfirstlane(item.split);
    // The split's steps of 32 tokens: of the history, then of the new rows that the tile's columns see.
    const int begin = split_begin(__builtin_amdgcn_readfirstlane(item.length), split, splits);
    const int end = split_begin(__builtin_amdgcn_readfirstlane(item.length), split + 1, splits);
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int i = lane & 15, g = lane >> 4;
    const int item_column = __builtin_amdgcn_readfirstlane(item.index) * kTile;
    const int column0 = item_column + wave * 16 * NT;
    const int history_steps = fp8_steps(history);
    const int old_end = min(end, history_steps);
    const int old_tokens = min(history, 32 * old_end);                   // of the history, tokens below this
    const int old_tiles = old_end > begin ? (old_end - begin + 1) / 2 : 0;
    const int seen_rows = min(rows, (item_column + kTile - 1) / group + 1);  // new rows that any column sees
    const int new_begin = 32 * (max(begin, history_steps) - history_steps);
    const int new_end = min(32 * (end - history_steps), seen_rows);
    const int new_tiles = new_end > new_begin ? (new_end - new_begin + kWideTokens - 1) / kWideTokens : 0;
    const int all_tiles = old_tiles + new_tiles;

    float* const entries = p.partials + ((int64_t)head * p.entries + __builtin_amdgcn_readfirstlane(item.entry)) * kEntry;

    U32x4 query[NT][kSteps];
    int seen[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int column = column0 + 16 * t + i;
        seen[t] = column < columns_in ? column / group : -1;
        const int row = column < columns_in ? column / group : 0;
        const uint16_t* q = p.query + (int64_t)(first + row) * p.query_stride +
                            ((int64_t)head * group + (column < columns_in ? column % group : 0)) * D;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const U32x4 a = *reinterpret_cast<const U32x4At8*>(q + 32 * s + 8 * g);
            query[t][s] = column < columns_in ? a : U32x4{0u, 0u, 0u, 0u};
        }
    }
    Fp8Columns<NT, kOut> columns;  // tile e: channels 16 e + 4 g + r
    columns.clear();
    const float to_log2 = p.softmax_scale * 1.44269504088896341f;
    const int page_shift = p.page_tokens == 16 ? 4 : 5;
    const int64_t plane_bytes = ((p.num_blocks * p.kv_heads) << page_shift) * D;

    // ---------------------------------------------------------------- fill
    // Thread `place` of a unit's 128: chunk place % kChunks of K token
    // place / kChunks; channels 4 (place % (D / 4)).. of V tokens
    // 4 (place / (D / 4))..  (D = 96: 96 of the 128.)
    const bool filler = (tid & 127) < 16 * kChunks;
    const int place = filler ? tid & 127 : 0;
    const int k_token = place / kChunks, k_chunk = place % kChunks;
    const int v_quad = place / (D / 4), v_word = place % (D / 4);
    // What a thread holds of a tile in flight: codes of the history, or new rows.
    struct Stage {
        U32x4 k[2];  // (codes: the first)
        U32x2 v[4];  // (codes: the first word)
        float key_scale, value_scale;
    };
    // (Not made uniform: a scalar load in flight would hold back every LDS wait.)
    const int unit = tid >> 7;
    // The table's entry for a tile's unit, unchecked; past the history the last one again.  (Loads
    // without a condition: behind one that a path leaves out, the wait is for all loads in flight.)
    auto entry_of = [&](int tile) {
        const int token = min(32 * begin + kWideTokens * tile + 16 * unit, old_tokens - 1);
        return p.block_table[(int64_t)request * p.block_table_stride + (token >> page_shift)];
    };
    int next_entry, stage_block;  // stage_block: -1 if no token of the unit counts
    auto fetch = [&](Stage& x, int tile) {
        if (tile >= old_tiles) {
            // New rows (clamped to the request's; what lies past them is masked).
            const int base = new_begin + kWideTokens * (tile - old_tiles) + 16 * unit;
            const uint16_t* k = p.key + (int64_t)(first + min(base + k_token, rows - 1)) * p.key_stride + (int64_t)head * D + 16 * k_chunk;
            x.k[0] = *reinterpret_cast<const U32x4At8*>(k);
            x.k[1] = *reinterpret_cast<const U32x4At8*>(k + 8);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x.v[r] = *reinterpret_cast<const U32x2*>(
                    p.value + (int64_t)(first + min(base + 4 * v_quad + r, rows - 1)) * p.value_stride + (int64_t)head * D + 4 * v_word);
            return;
        }
        const int token = 32 * begin + kWideTokens * tile + 16 * unit;
        const int block = token < old_tokens && next_entry >= 0 && next_entry < p.num_blocks ? next_entry : -1;
        const int64_t index = (int64_t)max(block, 0) * p.kv_heads + head;
        next_entry = entry_of(tile + 1);
        // (Without a block: the first one's bytes, of which no token counts.)
        x.key_scale = p.scales[index];
        x.value_scale = p.scales[index + p.num_blocks * p.kv_heads];
        const uint8_t* from = p.cache + ((index << page_shift) + (token & (p.page_tokens - 1))) * D;
        x.k[0] = *reinterpret_cast<const U32x4*>(from + k_token * D + 16 * k_chunk);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            x.v[r][0] = *reinterpret_cast<const uint32_t*>(from + plane_bytes + (4 * v_quad + r) * D + 4 * v_word);
        stage_block = block;
    };
    auto v_place = [&](WideTile<D>& tile, int channel, int unit, int quad) -> U32x2* {
        const int chunk = 4 * (unit >> 1) + quad;
        return reinterpret_cast<U32x2*>(&tile.v[channel][chunk ^ v_swizzle(channel)]) + (unit & 1);
    };
    auto store = [&](const Stage& x, int number) {
        WideTile<D>& tile = tiles[number & 1];
        bool odd = false;
        const int token = 16 * unit + k_token;
        if (number < old_tiles) {
            const int valid = stage_block >= 0 ? min(old_tokens - 32 * begin - kWideTokens * number - 16 * unit, 16) : 0;
            if (filler) {
                const U32x4 k = x.k[0];
                tile.k[token][(2 * k_chunk) ^ k_token] =
                    U32x4{bf16x2_of_fp8<false>(k[0]), bf16x2_of_fp8<true>(k[0]), bf16x2_of_fp8<false>(k[1]), bf16x2_of_fp8<true>(k[1])};
                tile.k[token][(2 * k_chunk + 1) ^ k_token] =
                    U32x4{bf16x2_of_fp8<false>(k[2]), bf16x2_of_fp8<true>(k[2]), bf16x2_of_fp8<false>(k[3]), bf16x2_of_fp8<true>(k[3])};
                // Slots past the history may hold NaN, which a weight of zero does not remove.
                uint32_t w[4], y[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = 4 * v_quad + r < valid ? x.v[r][0] : 0u;
                transpose_bytes(w, y);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *v_place(tile, 4 * v_word + c, unit, v_quad) = U32x2{bf16x2_of_fp8<false>(y[c]), bf16x2_of_fp8<true>(y[c])};
            }
            if ((tid & 127) == 0) {
                tile.key_scale[unit] = stage_block >= 0 ? factor_of_scores(x.key_scale, to_log2) : 1.f;
                tile.value_scale[unit] = stage_block >= 0 ? x.value_scale : 1.f;
                tile.valid[unit] = valid | (stage_block >= 0 && x.value_scale > kHugeScale ? kHugeFlag : 0);
            }
            return;
        }
        if (filler) {
            tile.k[token][(2 * k_chunk) ^ k_token] = x.k[0];
            tile.k[token][(2 * k_chunk + 1) ^ k_token] = x.k[1];
            // Infinities and NaN, which a weight of zero does not remove, and huge values are left out here and added apart.
            U32x2 w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    odd |= odd_bf16x2(x.v[r][h]);
                    w[r][h] = without_odd(x.v[r][h]);
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t pick = c & 1 ? 0x07060302u : 0x05040100u;
                *v_place(tile, 4 * v_word + c, unit, v_quad) =
                    U32x2{__builtin_amdgcn_perm(w[1][c >> 1], w[0][c >> 1], pick), __builtin_amdgcn_perm(w[3][c >> 1], w[2][c >> 1], pick)};
            }
        }
        if ((tid & 127) == 0) {
            tile.key_scale[unit] = to_log2;
            tile.value_scale[unit] = 1.f;
            tile.valid[unit] = 16;
        }
        if (odd) tile.odd = number;
    };

    // ---------------------------------------------------------------- products
    const bool idle = column0 >= columns_in;
    // The last new row of the split that the wave's columns see.
    const int new_last = min(new_end - 1, (column0 + 16 * NT - 1) / group);
    // (base: the tile's first new row, or -1 for the history.)
    auto compute = [&](int number) {
        WideTile<D>& tile = tiles[number & 1];
        const int base = number < old_tiles ? -1 : new_begin + kWideTokens * (number - old_tiles);
        if (base >= 0 && base > new_last) return;
#pragma unroll
        for (int st = 0; st < 2; ++st) {
            if (base >= 0 && base + 32 * st > new_last) break;
            float key_scale[2], value_scale[2];
            int valid[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                key_scale[u] = tile.key_scale[2 * st + u];
                value_scale[u] = tile.value_scale[2 * st + u];
                valid[u] = tile.valid[2 * st + u];
            }
            F32x4 dot[NT][2];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int u = 0; u < 2; ++u) dot[t][u] = F32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                U32x4 a[kSteps];
#pragma unroll
                for (int m = 0; m < kSteps; ++m) a[m] = tile.k[32 * st + 16 * u + i][(4 * m + g) ^ i];
#pragma unroll
                for (int m = 0; m < kSteps; ++m)
#pragma unroll
                    for (int t = 0; t < NT; ++t) dot[t][u] = mfma(a[m], query[t][m], dot[t][u]);
            }
            // V's operands arrive while the weights are computed.
            __builtin_amdgcn_sched_barrier(0);
            U32x4 operand[kOut];
#pragma unroll
            for (int e = 0; e < kOut; ++e) operand[e] = tile.v[16 * e + i][(4 * st + g) ^ v_swizzle(16 * e + i)];
            __builtin_amdgcn_sched_barrier(0);
            if (base < 0) {
                if (__builtin_amdgcn_readfirstlane((valid[0] ^ 16) | (valid[1] ^ 16)) != 0) {
                    if (__builtin_amdgcn_readfirstlane((valid[0] | valid[1]) & kHugeFlag) != 0) columns.make_room();
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                dot[t][u][r] = 4 * g + r < (valid[u] & (kHugeFlag - 1)) ? dot[t][u][r] : -__builtin_inff();
                }
            } else if (base + 32 * st + 31 > column0 / group || base + 32 * st + 31 >= new_end) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            dot[t][u][r] = base + 32 * st + 16 * u + 4 * g + r <= min(seen[t], new_end - 1) ? dot[t][u][r] : -__builtin_inff();
            }
            float weight[NT][2][4];
            U32x4 upper[NT][1], lower[NT][1];
            // (The wave that computes weights goes before one in its products: 105 -> 103 us for two chunks of 509 rows.)
            __builtin_amdgcn_s_setprio(2);
#pragma unroll
            for (int u = 0; u < 2; ++u) value_scale[u] *= columns.unit;
            fp8_softmax<NT, kOut, 2>(columns, dot, key_scale, value_scale, weight, upper, lower);
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int e = 0; e < kOut; ++e)
#pragma unroll
                for (int t = 0; t < NT; ++t) columns.out[t][e] = mfma(operand[e], upper[t][0], columns.out[t][e]);
#pragma unroll
            for (int e = 0; e < kOut; ++e)
#pragma unroll
                for (int t = 0; t < NT; ++t) columns.out[t][e] = mfma(operand[e], lower[t][0], columns.out[t][e]);
            if (base >= 0 && tile.odd == number) {
                // Huge values, infinities and NaN among the new ones, for the columns that see them.
                const float unit_of_weights = columns.unit;
                columns.make_room();
                for (int j = 0; j < 32; ++j) {
                    const int token = base + 32 * st + j;
                    if (token >= new_end) break;
                    const uint16_t* row = p.value + (int64_t)(first + token) * p.value_stride + (int64_t)head * D;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        // The weight (both its parts) of token j.
                        uint32_t up = 0, low = 0;
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                if (16 * u + 2 * x == (j & 18)) up = upper[t][0][2 * u + x], low = lower[t][0][2 * u + x];
                        if ((j & 1) == 0) up <<= 16, low <<= 16;
                        const float mine = __uint_as_float(up & 0xffff0000u) + __uint_as_float(low & 0xffff0000u);
                        const float w = __shfl(mine, i + 16 * ((j >> 2) & 3));
                        if (token > seen[t]) continue;
#pragma unroll
                        for (int e = 0; e < kOut; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const float x = bf16_f32(row[16 * e + 4 * g + r]);
                                if (!(fabsf(x) < kHugeValue)) columns.out[t][e][r] += w * (x * (columns.unit / unit_of_weights));
                            }
                    }
                }
            }
        }
    };

    Stage stage;
    next_entry = old_tiles > 0 ? entry_of(0) : -1;
    if (tid < 2) tiles[tid].odd = -1;
    __syncthreads();
    if (all_tiles > 0) {
        fetch(stage, 0);
        store(stage, 0);
        if (all_tiles > 1) fetch(stage, 1);
    }
    for (int n = 0; n < all_tiles; ++n) {
        __syncthreads();
        if (!idle) compute(n);
        if (n + 1 < all_tiles) store(stage, n + 1);
        if (n + 2 < all_tiles) fetch(stage, n + 2);
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        columns.sum[t] += __shfl_xor(columns.sum[t], 16);
        columns.sum[t] += __shfl_xor(columns.sum[t], 32);
    }

    // ---------------------------------------------------------------- finish
    const __amdgpu_buffer_rsrc_t handoff = handoff_resource(entries, (uint32_t)min((int64_t)columns_in * splits * kEntry * 4, (int64_t)0xfffffffc));
    auto output_row = [&](int column) {
        return p.output + (int64_t)(first + column / group) * p.output_stride + ((int64_t)head * group + column % group) * D;
    };
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int column = column0 + 16 * t + i;
        if (column >= columns_in) continue;
        if (splits == 1) {
            const float scale = join_scale(__float_as_uint(columns.marked_sum(t)), columns.sum[t]);
            uint16_t* out = output_row(column) + 4 * g;
#pragma unroll
            for (int e = 0; e < kOut; ++e) {
                const F32x4 o = columns.out[t][e] * scale;
                *reinterpret_cast<U32x2*>(out + 16 * e) = U32x2{bf16x2_rn(o[0], o[1]), bf16x2_rn(o[2], o[3])};
            }
            continue;
        }
        const uint32_t at = (uint32_t)(column * splits + split) * kEntry * 4;
#pragma unroll
        for (int e = 0; e < kOut; ++e) {
            const F32x4 o = columns.out[t][e];
            handoff_store4(handoff, at + 16 + 4 * (16 * e + 4 * g), o[0], o[1], o[2], o[3]);
        }
        if (g == 0) {
            handoff_store(handoff, at, columns.high[t]);
            handoff_store(handoff, at + 4, columns.marked_sum(t));
        }
    }
}

// The join of the wide kernel's parts, over the same plan: the workgroup of a
// split joins that share of its item's columns.  (The last of the splits alone
// would read 1 MB for 256 columns in 8 parts: one request of 2048 + 256 tokens
// took 68 us with that.)
template <int D>
__global__ __launch_bounds__(kWideThreads) void attention_fp8_join_kernel(const Fp8AttentionParams p) {
    constexpr int kTile = kWideTile, kEntry = D + 4;
    const int head = (int)(blockIdx.x % (unsigned)p.kv_heads);
    const PlanItem item = fp8_item<kTile>(p, (int)(blockIdx.x / (unsigned)p.kv_heads));
    const int request = __builtin_amdgcn_readfirstlane(item.request);
    const int splits = __builtin_amdgcn_readfirstlane(item.splits), split = __builtin_amdgcn_readfirstlane(item.split);
    if (request < 0 || splits == 1) return;
    const int group = p.heads / p.kv_heads;
    const int first = __builtin_amdgcn_readfirstlane(item.first), columns_in = __builtin_amdgcn_readfirstlane(item.rows);
    const int item_column = __builtin_amdgcn_readfirstlane(item.index) * kTile, count = min(kTile, columns_in - item_column);
    float* const entries = p.partials + ((int64_t)head * p.entries + __builtin_amdgcn_readfirstlane(item.entry)) * kEntry;
    const __amdgpu_buffer_rsrc_t handoff = handoff_resource(entries, (uint32_t)min((int64_t)columns_in * splits * kEntry * 4, (int64_t)0xfffffffc));
    fp8_join<D, kWideThreads, false>(handoff, item_column + count * split / splits, item_column + count * (split + 1) / splits, splits,
                              [&](int column) {
                                  return p.output + (int64_t)(first + column / group) * p.output_stride +
                                         ((int64_t)head * group + column % group) * D;
                              });
}

}  // namespace

hipError_t launch_quantize_fp8(const Fp8WriteParams& p, hipStream_t stream) {
    if (p.rows == 0 || p.requests == 0) return hipSuccess;
    const dim3 grid((unsigned)(p.rows / p.page_tokens + 2 * p.requests), (unsigned)((p.kv_heads + 3) / 4), 2), threads(256);
    if (p.head_dim == 128 && p.page_tokens == 16)
        hipLaunchKernelGGL((quantize_fp8_kernel<128, 16>), grid, threads, 0, stream, p);
    else if (p.head_dim == 128)
        hipLaunchKernelGGL((quantize_fp8_kernel<128, 32>), grid, threads, 0, stream, p);
    else if (p.page_tokens == 16)
        hipLaunchKernelGGL((quantize_fp8_kernel<96, 16>), grid, threads, 0, stream, p);
    else
        hipLaunchKernelGGL((quantize_fp8_kernel<96, 32>), grid, threads, 0, stream, p);
    return hipGetLastError();
}

namespace {

template <int D>
void launch_attention(const Fp8AttentionParams& p, hipStream_t stream) {
    const int64_t columns = p.rows * (p.heads / p.kv_heads);
    const int64_t items = p.items > 0 ? p.items : (columns / p.tile + p.requests) * p.splits;
    const dim3 grid((unsigned)(items * p.kv_heads)), threads(kStreamThreads);
    if (p.tile == 16)
        hipLaunchKernelGGL((attention_fp8_kernel<D, 1>), grid, threads, 0, stream, p);
    else if (p.tile == 32)
        hipLaunchKernelGGL((attention_fp8_kernel<D, 2>), grid, threads, 0, stream, p);
    else {
        hipLaunchKernelGGL((attention_fp8_wide_kernel<D>), grid, dim3(kWideThreads), 0, stream, p);
        if (p.splits > 1 || (p.items > 0 && p.plan_max_splits > 1))
            hipLaunchKernelGGL((attention_fp8_join_kernel<D>), grid, dim3(kWideThreads), 0, stream, p);
    }
}

}  // namespace

hipError_t launch_attention_fp8(const Fp8AttentionParams& p, hipStream_t stream) {
    if (p.rows == 0 || p.requests == 0) return hipSuccess;
    if (p.head_dim == 128)
        launch_attention<128>(p, stream);
    else
        launch_attention<96>(p, stream);
    return hipGetLastError();
}

}  // namespace rq
