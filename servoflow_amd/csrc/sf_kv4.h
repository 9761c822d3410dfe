// Layout of the 4-bit key / value cache, shared by its writer and readers.
//
// [B][H][blocks of 32 tokens], one block D * 36 contiguous bytes: key codes
// (16 D bytes), value codes (16 D bytes), key parameters and value parameters
// ([D / 64 groups][32 tokens] dwords each: step bf16, middle bf16 << 16).
//
// Key codes are the A operand of S^T = K Q^T: lane l = 16 g + r of a wave
// holds token r (tile 0) and 16 + r (tile 1), and of each group of 64
// channels the 16 channels 64 grp + 16 g .. + 15, 8 bytes: a 16-byte load is
// two tiles (D = 64) or two groups (D = 128).  Code e of a dword's 8 channels
// sits at nibble (e >> 1) + 4 (e & 1).
//
// Value codes are the A operand of O^T = V^T P^T, whose contraction runs over
// the block's 32 tokens in the order that S^T leaves in the registers: lane
// group g, element e is token 4 g + e (e < 4) or 16 + 4 g + e - 4.  Lane l
// holds channels 32 t + (l & 15) in the low and + 16 in the high nibbles,
// 8 bytes for each t, elements 0, 2, 1, 3 of a dword's four bytes.
// So a token owns whole bytes of each part, and appending one never reads.
#pragma once

#include <stdint.h>

namespace sfk {

constexpr int kKvBlock = 32;

__host__ __device__ inline int64_t kv4_blocks(int capacity) { return ((int64_t)capacity + kKvBlock - 1) / kKvBlock; }

// Byte offsets inside a block of head dim D.
template <int D>
struct Kv4 {
    static constexpr int kGroups = D / 64;
    static constexpr int kV = 16 * D;             // value codes
    static constexpr int kPar = 32 * D;           // key parameters
    static constexpr int kVPar = 34 * D;          // value parameters
    static constexpr int kBytes = 36 * D;

    // Dword of token `tok`'s key codes for channels 8 j .. 8 j + 7.
    __device__ static int key_dword(int tok, int j) {
        const int grp = j >> 3, g = (j >> 1) & 3, lane = 16 * g + (tok & 15), tile = tok >> 4;
        return D == 64 ? lane * 16 + tile * 8 + (j & 1) * 4 : tile * 1024 + lane * 16 + grp * 8 + (j & 1) * 4;
    }
    // Byte, from kV on, of token `tok`'s value codes of channels 32 t + dl (low nibble) and 32 t + 16 + dl (high).
    __device__ static int value_byte(int tok, int t, int dl) {
        const int g = (tok & 15) >> 2, e = tok & 3;
        return (t >> 1) * 1024 + (16 * g + dl) * 16 + (t & 1) * 8 + (tok >> 4) * 4 + ((e & 1) << 1 | e >> 1);
    }
    __device__ static int key_par(int tok, int grp) { return kPar + (grp * kKvBlock + tok) * 4; }
    __device__ static int value_par(int tok, int grp) { return kVPar + (grp * kKvBlock + tok) * 4; }
};

}  // namespace sfk
