// 16-bit numbers, eight or two at a time, for the kernels between the projections and attention.
#pragma once

#include "common.h"

namespace cozyq {

// Eight 16-bit elements as float32.
template <bool kHalf>
__device__ __forceinline__ void widen8(const i32x4& raw, float* v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = widen<kHalf>(static_cast<uint16_t>(static_cast<uint32_t>(raw[i / 2]) >> (16 * (i & 1))));
}

// The same where the type is known at run time alone: a branch, as a select would work out both.
__device__ __forceinline__ void widen8(const i32x4& raw, bool half, float* v) {
    if (half) {
        asm volatile("");
        widen8<true>(raw, v);
    } else {
        widen8<false>(raw, v);
    }
}

// Eight 16-bit elements at a 16-byte address, as float32.
template <bool kHalf>
__device__ __forceinline__ void load8(const uint16_t* p, float* v) {
    widen8<kHalf>(*reinterpret_cast<const i32x4*>(p), v);
}

// Two float32 values rounded to nearest even, the first in the low half: v_cvt_pk_bf16_f32 for bf16; for
// fp16 each float32 value stands on its own first (see narrow).
template <bool kHalf>
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
    if constexpr (kHalf) return narrow<true>(a) | (static_cast<uint32_t>(narrow<true>(b)) << 16);
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 two = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, two);
}

__device__ __forceinline__ uint32_t narrow2(float a, float b, bool half) {
    if (half) {
        asm volatile("");
        return narrow2<true>(a, b);
    }
    return narrow2<false>(a, b);
}

template <bool kHalf>
__device__ __forceinline__ void store8(uint16_t* p, const float* v) {
    i32x4 raw;
#pragma unroll
    for (int i = 0; i < 4; ++i) raw[i] = static_cast<int32_t>(narrow2<kHalf>(v[2 * i], v[2 * i + 1]));
    *reinterpret_cast<i32x4*>(p) = raw;
}

// Four 8-bit codes of a dword, int8 or E4M3, as float32 (exact).
template <bool kFp8>
__device__ __forceinline__ void codes4f(uint32_t c, float* v) {
    if constexpr (kFp8) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c), false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c), true);
        v[0] = lo[0];
        v[1] = lo[1];
        v[2] = hi[0];
        v[3] = hi[1];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>(c >> (8 * i)));
    }
}

}  // namespace cozyq
