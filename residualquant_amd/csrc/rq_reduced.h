// Launch parameters of the operators of a decode step at reduced precision
// (8-bit cache, 4-bit weights) and of its log probabilities, shared between
// the C ABI (capi.hip) and the kernels.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rq_plan.h"

namespace rq {

// Projections with 4-bit weights and group scales (linear_int4.hip).
constexpr int kLinearInt4MaxRows = 64;
struct Int4PackParams {
    const int8_t* codes;      // [out, in] in -8..7 with scales [out, in / group], or
    const uint16_t* scales;
    const uint16_t* weight;   // a BF16 weight [out, in] to quantize
    uint32_t* packed;
    uint16_t* packed_scales;
    int64_t out_features, in_features;
    int group;                // 32, 64 or 128; divides in_features
};
struct LinearInt4Params {
    const uint16_t* x;        // BF16 [rows, in]
    int64_t x_stride;
    const uint32_t* packed;
    const uint16_t* packed_scales;
    uint16_t* y;              // BF16 [rows, out]
    int64_t y_stride;
    int64_t rows, out_features, in_features;
    int group;
    int compute_units;        // of the launching device
    int chunk_blocks;         // set by the launch: blocks of 128 inputs of x in LDS at once
    bool aligned;             // set by the launch: 8-byte stores of y
};
size_t int4_code_bytes(int64_t out_features, int64_t in_features);
size_t int4_weight_bytes(int64_t out_features, int64_t in_features, int group);
hipError_t launch_pack_int4(const Int4PackParams& p, hipStream_t stream);
hipError_t launch_unpack_int4(const Int4PackParams& p, uint16_t* weight, hipStream_t stream);
hipError_t launch_linear_int4(const LinearInt4Params& p, hipStream_t stream);

// Log probabilities of given tokens (logprobs.hip).
constexpr int kLogprobMaxTop = 32;
struct LogprobParams {
    const void* logits;       // BF16 or FP32 [rows, vocab]
    int64_t stride;
    bool bf16;
    int64_t rows, vocab;
    const int64_t* tokens;    // [rows]
    float* logprob;           // [rows]
    float* entropy;           // [rows]
    int top;
    float* top_logprobs;      // [rows, top]
    int64_t* top_tokens;      // [rows, top]
};
hipError_t launch_logprobs(const LogprobParams& p, hipStream_t stream);

// Projections in 8-bit floating point with block scales (linear_fp8.hip).
constexpr int64_t kLinearFp8MaxRows = 1 << 20;
struct Fp8PackParams {
    const uint8_t* codes;     // E4M3 [out, in] with scales [out / 128, in / 128] (rounded up), or
    const void* scales;       // E8M0 bytes or FP32
    const uint16_t* weight;   // a BF16 weight [out, in] to quantize (E8M0 scales)
    uint8_t* packed;
    uint8_t* packed_scales;
    int64_t out_features, in_features;
    bool exponents;           // scales are E8M0
};
struct LinearFp8Params {
    const uint16_t* x;        // BF16 [rows, in]
    int64_t x_stride;
    const uint8_t* packed;
    const uint8_t* packed_scales;
    uint16_t* y;              // BF16 [rows, out]
    int64_t y_stride;
    int64_t rows, out_features, in_features;
    bool exponents;
    int compute_units;        // of the launching device
    uint8_t* x_codes;         // workspace: x in operand order
    uint32_t* x_scales;       // set by the launch: workspace [fours of blocks][tiles of 16 rows][16], four E8M0 bytes each
    bool wide;                // set by the launch: 16-byte loads of a few rows of x
};
size_t fp8_code_bytes(int64_t out_features, int64_t in_features);
size_t fp8_weight_bytes(int64_t out_features, int64_t in_features, bool exponents);
size_t linear_fp8_workspace(int64_t rows, int64_t in_features);
hipError_t launch_pack_fp8(const Fp8PackParams& p, hipStream_t stream);
hipError_t launch_unpack_fp8(const Fp8PackParams& p, uint16_t* weight, hipStream_t stream);
hipError_t launch_linear_fp8(const LinearFp8Params& p, hipStream_t stream);

// Rotation of a call's q and k, and K/V appended to a paged cache (rope_append.hip).
struct RopeAppendParams {
    const uint16_t* qkv;      // BF16 [rows, (heads + 2 kv_heads) D]
    int64_t qkv_stride;
    int64_t rows;
    int heads, kv_heads, head_dim, rotary;
    bool interleaved;
    const float* cos_table;   // [table_rows, rotary / 2]
    const float* sin_table;
    int64_t table_rows;
    const int64_t* positions; // [rows], or null: the tokens' places in their requests
    uint16_t* query;
    int64_t query_stride;
    uint16_t* key;
    int64_t key_stride;
    void* cache;              // [2, blocks, kv_heads, PT, D], E4M3 with scales or BF16
    float* scales;            // [2, blocks, kv_heads], null: BF16 pages
    int64_t num_blocks;
    int page_tokens;
    const int32_t* query_start_loc;
    const int32_t* seq_lens;
    int64_t requests;
    const int32_t* block_table;
    int64_t block_table_stride;
    int64_t max_pages;
    int span;                 // set by the launch: heads (q's, k's and v's in a row) per workgroup
};
hipError_t launch_rope_append(const RopeAppendParams& p, hipStream_t stream);

// Verification of drafted tokens (verify.hip).
struct VerifyParams {
    const void* target;       // BF16 or FP32 [rows, vocab]
    int64_t target_stride;
    const void* draft;        // as target, or null
    int64_t draft_stride;
    bool bf16;
    int64_t rows, vocab;
    const int64_t* tokens;    // [rows]
    const float* uniforms;    // [rows]
    const int32_t* query_start_loc;
    int64_t requests;
    int32_t* accepted;        // [requests]
    int64_t* out_tokens;      // [rows]
    int64_t chunks;           // of a row
    int each;                 // set by the launch: chunks per workgroup
    uint64_t* arrivals;       // workspace [requests] words of a cache line each, tagged arrival counts (rq_plan.h)
    double* sums;             // workspace [requests, chunks]
    uint64_t call_tag;        // of this call (48 bits, rq_plan.h)
};
constexpr int kVerifyArrivalStride = 16;  // words of 8 bytes
int64_t verify_chunks(int64_t requests, int64_t vocab, bool bf16);
hipError_t launch_verify(const VerifyParams& p, hipStream_t stream);

// Cache held in 8 bits (fp8_cache.hip): E4M3 codes [2, blocks, kv_heads, PT, D],
// FP32 scales [2, blocks, kv_heads].
struct Fp8WriteParams {
    const uint16_t* key;
    int64_t key_stride;
    const uint16_t* value;
    int64_t value_stride;
    int64_t rows;
    int kv_heads, head_dim;
    uint8_t* cache;
    float* scales;
    int64_t num_blocks;
    int page_tokens;
    const int32_t* query_start_loc;
    const int32_t* seq_lens;
    int64_t requests;
    const int32_t* block_table;
    int64_t block_table_stride;
    int64_t max_pages;
};
struct Fp8AttentionParams {
    const uint16_t* query;
    int64_t query_stride;
    const uint16_t* key;
    int64_t key_stride;
    const uint16_t* value;
    int64_t value_stride;
    uint16_t* output;
    int64_t output_stride;
    int64_t rows;
    int heads, kv_heads, head_dim;
    const uint8_t* cache;
    const float* scales;
    int64_t num_blocks;
    int page_tokens;
    const int32_t* query_start_loc;
    const int32_t* seq_lens;
    int64_t requests;
    const int32_t* block_table;
    int64_t block_table_stride;
    int64_t max_pages;
    float softmax_scale;
    // Work plan (rq_plan.h).  A request's rows x group query heads per K/V
    // head are its columns, in tiles of `tile`; its history and new rows are
    // read in steps of 32 tokens.  Up to kPlanRequests requests, `items`
    // workgroups per K/V head are planned on the device; with more (items 0)
    // every tile takes `splits`.
    int tile;                 // 16, 32 or 256 columns per workgroup
    int items;
    int splits;               // of every tile of equal requests
    int plan_target, plan_min, plan_max_splits;  // PlanSizes, in steps
    int64_t entries;          // partials per K/V head
    float* partials;          // workspace [kv_heads, entries, D + 4]
    uint64_t call_tag;        // of this call (48 bits, rq_plan.h)
};
__host__ __device__ __forceinline__ PlanSizes fp8_sizes(const Fp8AttentionParams& p) {
    return PlanSizes{p.plan_target, p.splits, p.plan_min, 1 << 24, p.plan_max_splits, 0, 1, 9, 0};
}
hipError_t launch_quantize_fp8(const Fp8WriteParams& p, hipStream_t stream);
hipError_t launch_attention_fp8(const Fp8AttentionParams& p, hipStream_t stream);

}  // namespace rq
