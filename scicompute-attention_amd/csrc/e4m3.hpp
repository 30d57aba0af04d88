// The 8-bit form of K and V in a paged cache, and its conversions.
//
// Of the D values x of one token and KV head, with a = max |x|, k is the least integer, at least
// -126, with a <= 448 * 2^k (448 is the largest e4m3 value). x is held as the e4m3 value (4
// significant bits, smallest step 2^-9) nearest to x / 2^k, ties to even, and the row's k as the
// byte k + 127. A row that was never written holds zeros and the byte 0.
//
// Why a power of two: x / 2^k and code * 2^k are exact, so that a code does not depend on how a
// division rounds, and every product code * 2^k is itself a number of the 16-bit type: attention
// over 8-bit pages is attention over 16-bit values, converted in registers with no rounding of its
// own. An e4m3 value has as many bits whatever its size, so that only values below about 2^-14 of
// the row's largest notice the coarser scale.
//
// Magnitudes above 1.875 times the type's largest power of two (61440 in fp16) would round to the
// next power of two, which the type does not have: they are held as that value (off by less than
// the 2^-4 that any value may be), infinities too. NaN is held as NaN and does not count for a.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sca_device.hpp"

namespace sca_hip {
namespace {

template <typename E>
struct Held;  // conversions of one 16-bit type

template <>
struct Held<F16> {
    static constexpr float kLargest = 61440.0f;
    // Codes 2 * half and 2 * half + 1 of the word times `unit` (a power of two), as a packed pair.
    template <bool kHalf>
    static __device__ __forceinline__ uint32_t widen2(uint32_t codes, float unit) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, unit, kHalf));
    }
};

template <>
struct Held<BF16> {
    static constexpr float kLargest = 0x1.ep127f;
    template <bool kHalf>
    static __device__ __forceinline__ uint32_t widen2(uint32_t codes, float unit) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, unit, kHalf));
    }
};

// Four codes of a word -> two packed pairs; eight -> an MFMA fragment's 16 bytes.
template <typename E>
__device__ __forceinline__ uint2 Widen4(uint32_t codes, float unit) {
    return make_uint2(Held<E>::template widen2<false>(codes, unit),
                      Held<E>::template widen2<true>(codes, unit));
}
template <typename E>
__device__ __forceinline__ uint4 Widen8(uint32_t lo, uint32_t hi, float unit) {
    const uint2 a = Widen4<E>(lo, unit), b = Widen4<E>(hi, unit);
    return make_uint4(a.x, a.y, b.x, b.y);
}

// 2^k of the byte k + 127 (0: a row never written, whose codes are zeros too).
__device__ __forceinline__ float UnitOf(uint32_t exponent) {
    return __builtin_bit_cast(float, exponent << 23);
}

// The byte k + 127 of a row with largest magnitude a (finite, not above Held::kLargest): 448 is
// 1.75 * 2^8, so k is a's exponent less 8, and one more past a mantissa of 1.75.
__device__ __forceinline__ uint32_t ExponentFor(float a) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, a);
    const int k = static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return static_cast<uint32_t>(k < 1 ? 1 : k);
}
// 2^-k of the byte k + 127, which is at least 1 and, as k <= 120, never above 247.
__device__ __forceinline__ float InverseUnit(uint32_t exponent) {
    return __builtin_bit_cast(float, (254u - exponent) << 23);
}

// Four values (already divided by 2^k, at most 448) -> a word of codes, ties to even.
__device__ __forceinline__ uint32_t Codes4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return static_cast<uint32_t>(w);
}

}  // namespace
}  // namespace sca_hip
