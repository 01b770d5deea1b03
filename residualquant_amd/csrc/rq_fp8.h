// What the writers of pages held in 8 bits share (fp8_cache.hip,
// rope_append.hip): one wave per (page, head, plane), the page's new values in
// its registers.
#pragma once

#include "rq_device.h"

namespace rq {

typedef uint32_t U32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t U32x2 __attribute__((ext_vector_type(2)));
typedef U32x4 U32x4At8 __attribute__((aligned(8)));  // 16 bytes on an 8-byte boundary

// Chunks of 8 values of a page that a lane holds: chunk 64 c + lane of its rows.
template <int D, int PT>
constexpr int kPageChunks = (PT * (D / 8) + 63) / 64;

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

// Four E4M3 codes of two words of two BF16 values over a power of two, |x| <= 448 of
// it: what fp8x4_rn makes of the quotients, infinities and NaN included (checked on the
// device for all values at powers from 2^-126 to 2^120), without unpacking them.
__device__ __forceinline__ uint32_t fp8x4_of_bf16(uint32_t low, uint32_t high, float scale) {
    typedef __bf16 Bf16x2 __attribute__((ext_vector_type(2)));
    typedef short I16x2 __attribute__((ext_vector_type(2)));
    I16x2 codes = {0, 0};
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(codes, __builtin_bit_cast(Bf16x2, low), scale, false);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(codes, __builtin_bit_cast(Bf16x2, high), scale, true);
    return __builtin_bit_cast(uint32_t, codes);
}

// The larger sizes of pairs of BF16 values, as bits (infinities and NaN are the largest).
__device__ __forceinline__ uint32_t larger_sizes(uint32_t a, uint32_t b) {
    typedef uint16_t U16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(U16x2, a), __builtin_bit_cast(U16x2, b)));
}
constexpr uint32_t kBf16Infinity = 0x7f80u;
// A pair's sizes, 0 in the place of what is not finite.
__device__ __forceinline__ uint32_t finite_sizes(uint32_t x) {
    x &= 0x7fff7fffu;
    return ((x & 0xffffu) < kBf16Infinity ? x & 0xffffu : 0u) | (x < (kBf16Infinity << 16) ? x & 0xffff0000u : 0u);
}

__device__ __forceinline__ bool power_of_two(float x) { return (__float_as_uint(x) & 0x7fffffu) == 0; }

// (Two values per instruction, maximum and conversion alike, leave a page of 32 rows
// of 128 channels 124 registers in place of 166.)  A page's rows from `slot` on from `values` (zeros where there are none), its scale, and where that grows its
// earlier rows once more.  place(c): which chunk of the new rows values[c] is, -1: none.
template <int D, int PT, int Held, class Place>
__device__ __forceinline__ void write_fp8_page(const U32x4 (&values)[Held], uint8_t* codes, float* page_scale, float before,
                                               int slot, Place place) {
    constexpr int kRow = D / 8, kChunks = kPageChunks<D, PT>;
    const int lane = threadIdx.x & 63;
    auto largest_of = [&](bool finite) {
        uint32_t most = 0;
#pragma unroll
        for (int c = 0; c < Held; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                most = larger_sizes(most, finite ? finite_sizes(values[c][e]) : values[c][e] & 0x7fff7fffu);
        most = max(most >> 16, most & 0xffffu);
#pragma unroll
        for (int d = 32; d; d >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d));
        return most;
    };
    uint32_t most = largest_of(false);
    if (most >= kBf16Infinity) most = largest_of(true);  // (the same for all lanes)
    const float largest = __uint_as_float(most << 16);
    const float need = needed_scale(largest);
    const float scale = slot > 0 && before >= need ? before : need;

    if (slot > 0 && scale > before) {
        const float shrink = before / scale;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int chunk = 64 * c + lane;
            if (chunk >= slot * kRow) continue;
            U32x2* held = reinterpret_cast<U32x2*>(codes) + chunk;
            U32x2 word = *held;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(word[w], false), high = __builtin_amdgcn_cvt_pk_f32_fp8(word[w], true);
                word[w] = fp8x4_rn(low[0] * shrink, low[1] * shrink, high[0] * shrink, high[1] * shrink);
            }
            *held = word;
        }
    }
    // (A scale that the caller made may be any number.)
    const bool exact = power_of_two(scale) && scale <= 0x1p120f;
#pragma unroll
    for (int c = 0; c < Held; ++c) {
        const int chunk = place(c);
        if (chunk < 0) continue;
        U32x2 word;
        if (exact) {
            word = U32x2{fp8x4_of_bf16(values[c][0], values[c][1], scale), fp8x4_of_bf16(values[c][2], values[c][3], scale)};
        } else {
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[2 * e] = __uint_as_float(values[c][e] << 16) / scale;
                x[2 * e + 1] = __uint_as_float(values[c][e] & 0xffff0000u) / scale;
            }
            word = U32x2{fp8x4_rn(x[0], x[1], x[2], x[3]), fp8x4_rn(x[4], x[5], x[6], x[7])};
        }
        reinterpret_cast<U32x2*>(codes)[slot * kRow + chunk] = word;
    }
    if (lane == 0) *page_scale = scale;
}

}  // namespace rq
