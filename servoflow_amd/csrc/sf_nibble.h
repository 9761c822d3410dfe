// 4-bit codes as matrix operands, shared by the 4-bit weights and the 4-bit
// key / value cache.
#pragma once

#include "sf_device.h"

namespace sfk {

// Makes the compiler hold a constant in a register: v_and_or_b32 takes no two
// literals, and from two it makes a v_and and a v_or (a third instruction for
// each pair of codes).
struct NibbleMask {
    uint32_t mask;   // the nibble's place in both halves
    uint32_t base;   // 16.0 in both halves
};
template <bool F16>
__device__ __forceinline__ NibbleMask nibble_mask() {
    NibbleMask m = {F16 ? 0x03C003C0u : 0x00780078u, F16 ? 0x4C004C00u : 0x41804180u};
    asm("" : "+v"(m.mask));
    asm("" : "+s"(m.base));
    return m;
}

// The codes c at nibbles (n, n + 4) of w, n = 0..3, as the pair (16 + c,
// 16 + c') of 16-bit floats: the nibble becomes the top of 16.0's mantissa.
template <bool F16, int n>
__device__ __forceinline__ uint32_t nibble_pair_plus16(uint32_t w, NibbleMask m) {
    constexpr int sh = 4 * n - (F16 ? 6 : 3);
    const uint32_t v = sh < 0 ? w << (sh < 0 ? -sh : 0) : w >> (sh < 0 ? 0 : sh);
    return (v & m.mask) | m.base;
}

template <bool F16>
__device__ __forceinline__ u32x4 nibbles_plus16(uint32_t w, NibbleMask m) {
    return u32x4{nibble_pair_plus16<F16, 0>(w, m), nibble_pair_plus16<F16, 1>(w, m), nibble_pair_plus16<F16, 2>(w, m),
                 nibble_pair_plus16<F16, 3>(w, m)};
}

// mfma16x16x32 on operands given as bits.
template <bool F16>
__device__ __forceinline__ f32x4 mfma_16b(u32x4 a, u32x4 b, f32x4 c) {
    return F16 ? mfma16x16x32_f16(u32x4_as_f16x8(a), u32x4_as_f16x8(b), c)
               : mfma16x16x32(u32x4_as_bf16x8(a), u32x4_as_bf16x8(b), c);
}

}  // namespace sfk
