// 4-bit codes as matrix operands, shared by the 4-bit weights and the 4-bit
// key / value cache.
#pragma once

#include "sf_device.h"

namespace sfk {

// The codes c at nibbles (n, n + 4) of w, n = 0..3, as the pair (16 + c,
// 16 + c') of 16-bit floats: the nibble becomes the top of 16.0's mantissa.
template <bool F16, int n>
__device__ __forceinline__ uint32_t nibble_pair_plus16(uint32_t w) {
    constexpr int sh = 4 * n - (F16 ? 6 : 3);
    const uint32_t v = sh < 0 ? w << (sh < 0 ? -sh : 0) : w >> (sh < 0 ? 0 : sh);
    return F16 ? (v & 0x03C003C0u) | 0x4C004C00u : (v & 0x00780078u) | 0x41804180u;
}

template <bool F16>
__device__ __forceinline__ u32x4 nibbles_plus16(uint32_t w) {
    return u32x4{nibble_pair_plus16<F16, 0>(w), nibble_pair_plus16<F16, 1>(w), nibble_pair_plus16<F16, 2>(w),
                 nibble_pair_plus16<F16, 3>(w)};
}

// mfma16x16x32 on operands given as bits.
template <bool F16>
__device__ __forceinline__ f32x4 mfma_16b(u32x4 a, u32x4 b, f32x4 c) {
    return F16 ? mfma16x16x32_f16(u32x4_as_f16x8(a), u32x4_as_f16x8(b), c)
               : mfma16x16x32(u32x4_as_bf16x8(a), u32x4_as_bf16x8(b), c);
}

}  // namespace sfk
