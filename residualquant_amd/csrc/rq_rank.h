// Order of logits and of (logit, index) pairs as unsigned integers, for the
// device and for checks on the host.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rq {

// Order of values as numbers: -0 and +0 alike, NaN above all.  (Not by 32 set bits: the key of a NaN
// at index 0 would be kAboveKeys.)
__host__ __device__ __forceinline__ uint32_t ordered_bits(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x != x ? 0xfffffffeu : (u >> 31) ? ~u : u | 0x80000000u;
}

// Order of (value, index): equal values by the lower index.
__host__ __device__ __forceinline__ uint64_t rank_key(float x, uint32_t index) {
    return ((uint64_t)ordered_bits(x) << 32) | (0xffffffffu - index);
}

// Above every key.
constexpr uint64_t kAboveKeys = ~0ull;

// The larger of `best` and a key that lies below `below`: the step of a pass for the next alternative.
__host__ __device__ __forceinline__ uint64_t next_rank(uint64_t best, uint64_t key, uint64_t below) {
    return key < below && key > best ? key : best;
}

}  // namespace rq
