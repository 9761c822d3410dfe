// Per-head RMSNorm of queries and keys with the position rotation in the same
// pass, into tensors or into the 4-bit key / value cache, and the cache's
// read-back (gfx950).
//
// The split + q_norm / k_norm of the reference's attention layers
// (split_ops.cuh:62-84, dit_block.cu:185-196, 262-272) for head dims 64 and
// 128 and key heads shared by query heads; the reference has no rotation and
// caches nothing.
//
// D / 8 lanes hold a head row, 8 channels each, so a row's sum of squares is
// three or four DPP steps and the rotation's partner in the "halves" pairing
// one cross-lane move.  Each row is read once and written once: the bound is
// the copy rate.  The angle's fraction of a turn is formed in 64 bits,
// position * inv_freq / 2 pi, so a position of 2^31 keeps 20 bits of it; sine
// and cosine of the remaining half turn are 32-bit.  They depend on the token
// alone: a workgroup computes them once per token into LDS for all its heads.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "sf_device.h"
#include "sf_hip.h"
#include "sf_kv4.h"

namespace sfk {

constexpr int kRopeTokens = kKvBlock;   // tokens of a workgroup, at most

struct RopeArgs {
    const void* src[3];
    int64_t ss[3][3];
    void* out[3];
    int64_t os[3][3];
    const float* gamma[2];
    const int32_t* positions;
    const int32_t* slots;
    const double* inv_freq;
    uint8_t* cache;
    int64_t cache_blocks;   // per (b, h)
    int heads[3];
    int S, cap, rot, interleaved, in_kind, out_kind;
    float eps;
    int tok_per_wg, windows;           // a batch element's tokens in windows
    int heads_per_wg;
    int heads_magic;                   // ceil(2^16 / heads_per_wg): (i * this) >> 16 is i / heads_per_wg, i < 2048
};

// kind: 0 fp32, 1 bf16, 2 fp16
__device__ __forceinline__ void load8(const void* p, int64_t at, int kind, float v[8]) {
    if (kind == 0) {
        const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
        const f32x4 a = q[0], b = q[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
        return;
    }
    const u32x4 r = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t u = r[e];
        if (kind == 1) {
            v[2 * e] = __uint_as_float(u << 16);
            v[2 * e + 1] = __uint_as_float(u & 0xffff0000u);
        } else {
            v[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)u);
            v[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
        }
    }
}

__device__ __forceinline__ void store8(void* p, int64_t at, int kind, const float v[8]) {
    if (kind == 0) {
        f32x4* q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + at);
        q[0] = f32x4{v[0], v[1], v[2], v[3]};
        q[1] = f32x4{v[4], v[5], v[6], v[7]};
        return;
    }
    u32x4 u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        u[e] = kind == 1 ? pack_bf16x2(v[2 * e], v[2 * e + 1]) : pack_f16x2_rn(v[2 * e], v[2 * e + 1]);
    *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at) = u;
}

// max over the 8 lanes of half a DPP row (row8_sum's steps).
__device__ __forceinline__ float row8_max(float x) {
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, true)));
    x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, true)));
    return fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xF, 0xF, true)));
}
__device__ __forceinline__ uint32_t row8_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xF, 0xF, true));
    x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xF, 0xF, true));
    return max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, true));
}

// Step and middle of a group of 64 channels held by 8 lanes, and the lane's
// eight codes, channel e at nibble (e >> 1) + 4 (e & 1).  The step is a power of
// two times a bf16, so t * step is exact for the whole t next to the approximate
// quotient, and comparing with it gives the floor of the exact quotient.
__device__ __forceinline__ uint32_t kv4_quantise(const float v[8], uint32_t* par) {
    float mx = v[0], mn = -v[0];
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        mx = fmaxf(mx, v[e]);
        mn = fmaxf(mn, -v[e]);
        big = max(big, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    mx = row8_max(mx);
    mn = -row8_max(mn);
    if (row8_max(big) >= 0x7f800000u) {   // an infinity or a NaN: the group reads back as NaN
        *par = 0x7fc07fc0u;
        return 0;
    }
    // fp32's last few numbers would round to an infinity
    const uint32_t mid_bits = f32_to_bf16_bits(__builtin_amdgcn_fmed3f(0.5f * mx + 0.5f * mn, -0x1.fep127f, 0x1.fep127f));
    const float mid = bf16_bits_to_f32(mid_bits);
    const float a = fmaxf(mx - mid, mid - mn);
    const uint32_t up = min((__float_as_uint(a) + 0xffffu) & 0xffff0000u, 0x7f7f0000u);   // bf16's largest at most
    float s = __uint_as_float(up) * 0.125f;
    if (s < 1.1754944e-38f) s = 0.f;   // below the normal range: every code stands for the middle
    *par = __float_as_uint(s) >> 16 | mid_bits << 16;
    if (s == 0.f) return 0x88888888u;
    const float inv = __builtin_amdgcn_rcpf(s);
    uint32_t c = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float d = v[e] - mid, t = rintf(d * inv);
        const int n = (int)t + (d < t * s ? 7 : 8);
        c |= (uint32_t)min(max(n, 0), 15) << (4 * ((e >> 1) + 4 * (e & 1)));
    }
    return c;
}

// A lane's codes of token `tok` to `codes`, the start of its head's key or value
// codes, with the parameters `par_at` bytes on.  Inlined with a pointer that is
// known to be of global memory or of LDS: one that may be either would be
// addressed by flat instructions, which tell the two apart by the address before
// the instruction's own offset is added.
template <int D, typename P>
__device__ __forceinline__ void kv4_put(P codes, int par_at, int tok, bool value, int j, uint32_t c, uint32_t other,
                                        uint32_t par) {
    if ((j & 7) == 0) *reinterpret_cast<uint32_t*>(codes + par_at + ((j >> 3) * kKvBlock + tok) * 4) = par;
    if (!value) {
        *reinterpret_cast<uint32_t*>(codes + Kv4<D>::key_dword(tok, j)) = c;
        return;
    }
    // Lanes j and j ^ 2 hold channels 16 apart, the low and the high halves of eight bytes: the first writes those of
    // channels 0, 4, 1, 5, as its nibbles lie, the other 2, 6, 3, 7.
    const bool hi = j & 2;
    const uint32_t w = hi ? (other >> 4 & 0x0f0f0f0fu) | (c & 0xf0f0f0f0u) : (c & 0x0f0f0f0fu) | (other << 4 & 0xf0f0f0f0u);
    P to = codes + Kv4<D>::value_byte(tok, j >> 2, 8 * (j & 1) + (hi ? 2 : 0));
    to[0] = (uint8_t)w;
    to[4 * 16] = (uint8_t)(w >> 8);
    to[16] = (uint8_t)(w >> 16);
    to[5 * 16] = (uint8_t)(w >> 24);
}

// One workgroup: up to tok_per_wg tokens of a batch element and heads_per_wg of
// the query, key and value heads in a row.  Into a cache the windows of tokens
// follow the cache's blocks, as far as the slots count up from the element's
// first one: a window of 32 tokens that fills a block is put together in LDS
// and stored as it lies there, 16 bytes a lane; other tokens are stored piece by
// piece (a token's codes are 4-byte and 1-byte pieces of its block: 4374 tokens
// of 32 heads took 45 us that way).
template <int D, bool CACHE>
__global__ __launch_bounds__(256) void heads_rope_kernel(const RopeArgs p) {
    constexpr int L = D / 8, kRows = 256 / L;
    constexpr int kImage = 16 * D + 2 * D;                  // a head's codes and parameters of 32 tokens, keys or values
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float2* cs = reinterpret_cast<float2*>(lds);                                      // [tok_per_wg][rot / 2]
    uint8_t* image = lds + sizeof(float2) * (size_t)p.tok_per_wg * (p.rot >> 1);      // [heads_per_wg][kImage]
    __shared__ int tpos[kRopeTokens], tslot[kRopeTokens], odd;
    __shared__ __attribute__((aligned(16))) float gamma[2][D];
    const int b = blockIdx.x / p.windows, win = blockIdx.x % p.windows;
    const int64_t m0 = (int64_t)b * p.S;
    int s0 = win * p.tok_per_wg, s1 = min(s0 + p.tok_per_wg, p.S);
    const int32_t* slots = p.slots ? p.slots : p.positions;
    if (CACHE && p.tok_per_wg == kKvBlock) {
        const int off = slots ? slots[m0] & (kKvBlock - 1) : 0;
        s1 = min(s0 + kKvBlock - off, p.S);   // the last window ends at S or behind it
        s0 = max(s0 - off, 0);
    }
    const int nt = s1 - s0, half = p.rot >> 1;
    if (nt <= 0) return;
    if (threadIdx.x == 0) odd = nt != kKvBlock;
    if (threadIdx.x < 2 * D && p.gamma[threadIdx.x / D]) gamma[threadIdx.x / D][threadIdx.x % D] = p.gamma[threadIdx.x / D][threadIdx.x % D];
    __syncthreads();
    if ((int)threadIdx.x < nt) {
        const int s = s0 + (int)threadIdx.x, pos = p.positions ? p.positions[m0 + s] : s;
        const int slot = slots ? slots[m0 + s] : s;
        tpos[threadIdx.x] = pos;
        tslot[threadIdx.x] = slot;
        const int first = slots ? slots[m0 + s0] : s0;
        if (CACHE && (pos < 0 || first < 0 || (first & (kKvBlock - 1)) || slot != first + (int)threadIdx.x || slot >= p.cap))
            odd = 1;
    }
    __syncthreads();
    const bool whole = CACHE && !odd;
    for (int i = threadIdx.x; i < nt * half; i += 256) {
        const double turns = (double)tpos[i / half] * (p.inv_freq[i % half] * 0.15915494309189533577);
        float c, s;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        cs[i] = float2{c, s};
    }
    __syncthreads();

    const int j = threadIdx.x & (L - 1), sub = threadIdx.x / L;
    const int h0 = blockIdx.y * p.heads_per_wg;
    const int nh = min(p.heads_per_wg, p.heads[0] + p.heads[1] + p.heads[2] - h0);
    const int rows = nt * p.heads_per_wg;
    for (int i = sub; i < rows; i += kRows) {
        const int ti = (i * p.heads_magic) >> 16, hi = i - ti * p.heads_per_wg;
        if (hi >= nh || tpos[ti] < 0) continue;   // whole groups of L lanes; a padding token is not written
        int h = h0 + hi, sec = 0;
        if (h >= p.heads[0]) h -= p.heads[0], sec = 1;
        if (sec == 1 && h >= p.heads[1]) h -= p.heads[1], sec = 2;
        float v[8];
        load8(p.src[sec], b * p.ss[sec][0] + h * p.ss[sec][1] + (s0 + ti) * p.ss[sec][2] + 8 * j, p.in_kind, v);
        if (sec == 0 ? p.gamma[0] != nullptr : sec == 1 && p.gamma[1]) {
            float q = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) q += v[e] * v[e];
            q = L == 8 ? row8_sum(q) : row16_sum(q);
            const float r = __builtin_amdgcn_rsqf(q * (1.f / (float)D) + p.eps);   // one unit
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = v[e] * r * gamma[sec][8 * j + e];
        }
        if (sec < 2 && half) {
            const float2* t = cs + ti * half;
            if (p.interleaved) {
                if (8 * j < p.rot) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 w = t[4 * j + e];
                        const float x = v[2 * e], y = v[2 * e + 1];
                        v[2 * e] = x * w.x - y * w.y;
                        v[2 * e + 1] = y * w.x + x * w.y;
                    }
                }
            } else {   // the partner's 8 channels are rot / 16 lanes away
                const int step = p.rot >> 4;
                const bool low = j < step, in = j < 2 * step;
                const int lane = (int)(threadIdx.x & 63);
                const int from = in ? (low ? lane + step : lane - step) : lane;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float y = __shfl(v[e], from, 64);
                    if (in) {
                        const float2 w = t[8 * (low ? j : j - step) + e];
                        v[e] = low ? v[e] * w.x - y * w.y : v[e] * w.x + y * w.y;
                    }
                }
            }
        }
        if (sec == 0 || !CACHE) {
            store8(p.out[sec], b * p.os[sec][0] + h * p.os[sec][1] + (s0 + ti) * p.os[sec][2] + 8 * j, p.out_kind, v);
            continue;
        }
        if constexpr (CACHE) {
            uint32_t par;
            const uint32_t c = kv4_quantise(v, &par);
            const uint32_t other = (uint32_t)__shfl_xor((int)c, 2, 64);
            const int slot = tslot[ti];
            if (slot < 0 || slot >= p.cap) continue;
            const int tok = slot % kKvBlock;
            if (whole) {   // the head's image in LDS: codes, then parameters
                const int head = (sec == 1 ? p.heads[0] + h : p.heads[0] + p.heads[1] + h) - h0;
                kv4_put<D>(image + head * kImage, 16 * D, tok, sec == 2, j, c, other, par);
            } else {
                uint8_t* blk = p.cache + (((int64_t)b * p.heads[1] + h) * p.cache_blocks + slot / kKvBlock) * Kv4<D>::kBytes;
                if (sec == 1) kv4_put<D>(blk, Kv4<D>::kPar, tok, false, j, c, other, par);
                else kv4_put<D>(blk + Kv4<D>::kV, Kv4<D>::kVPar - Kv4<D>::kV, tok, true, j, c, other, par);
            }
        }
    }
    if constexpr (CACHE) {
        if (!whole) return;
        __syncthreads();
        constexpr int kPieces = kImage / 16, kCodes = 16 * D / 16;
        for (int i = threadIdx.x; i < nh * kPieces; i += 256) {
            const int hi = i / kPieces, piece = i % kPieces, g = h0 + hi - p.heads[0];
            if (g < 0) continue;   // a query head
            const bool val = g >= p.heads[1];
            const int h = val ? g - p.heads[1] : g;
            uint8_t* blk = p.cache + (((int64_t)b * p.heads[1] + h) * p.cache_blocks + tslot[0] / kKvBlock) * Kv4<D>::kBytes;
            const int to = piece < kCodes ? (val ? Kv4<D>::kV : 0) + 16 * piece
                                          : (val ? Kv4<D>::kVPar : Kv4<D>::kPar) + 16 * (piece - kCodes);
            *reinterpret_cast<u32x4*>(blk + to) = *reinterpret_cast<const u32x4*>(image + hi * kImage + 16 * piece);
        }
    }
}

// Eight channels of a token's key (sec 0) or value out of its block (in global
// memory or in LDS: see kv4_put).
template <int D, typename P>
__device__ __forceinline__ void kv4_get(P blk, int tok, int sec, int j, float v[8]) {
    const uint32_t par = *reinterpret_cast<const uint32_t*>(
        blk + (sec ? Kv4<D>::value_par(tok, j >> 3) : Kv4<D>::key_par(tok, j >> 3)));
    const float st = __uint_as_float(par << 16), mid = __uint_as_float(par & 0xffff0000u);
    if (sec) {
        P from = blk + Kv4<D>::kV + Kv4<D>::value_byte(tok, j >> 2, 8 * (j & 1));
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = __builtin_fmaf((float)((uint32_t)from[16 * e] >> (j & 2 ? 4 : 0) & 15u) - 7.5f, st, mid);
    } else {
        const uint32_t c = *reinterpret_cast<const uint32_t*>(blk + Kv4<D>::key_dword(tok, j));
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf((float)(c >> (4 * ((e >> 1) + 4 * (e & 1))) & 15u) - 7.5f, st, mid);
    }
}

struct Kv4ReadArgs {
    const uint8_t* cache;
    int64_t cache_blocks;
    const int32_t* slots;
    void* out[2];
    int64_t os[2][3];
    int H, S, cap, out_kind, windows;
};

constexpr int kReadHeads = 4;   // heads of a workgroup

// The values of given slots, 32 tokens of four heads to a workgroup.  Tokens
// that fill a block are read through LDS, whole blocks at 16 bytes a lane; others
// piece by piece.
template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4ReadArgs p) {
    constexpr int L = D / 8, kRows = 256 / L, kBlk = Kv4<D>::kBytes;
    __shared__ __attribute__((aligned(16))) uint8_t image[kReadHeads * kBlk];
    __shared__ int tslot[kKvBlock], odd;
    const int b = blockIdx.x / p.windows, win = blockIdx.x % p.windows, h0 = blockIdx.y * kReadHeads;
    const int nh = min(kReadHeads, p.H - h0);
    const int64_t m0 = (int64_t)b * p.S;
    const int off = p.slots ? p.slots[m0] & (kKvBlock - 1) : 0;
    const int s0 = max(win * kKvBlock - off, 0), s1 = min((win + 1) * kKvBlock - off, p.S), nt = s1 - s0;
    if (nt <= 0) return;
    if (threadIdx.x == 0) odd = nt != kKvBlock;
    __syncthreads();
    if ((int)threadIdx.x < nt) {
        const int s = s0 + (int)threadIdx.x, slot = p.slots ? p.slots[m0 + s] : s, first = p.slots ? p.slots[m0 + s0] : s0;
        tslot[threadIdx.x] = slot;
        if (first < 0 || (first & (kKvBlock - 1)) || slot != first + (int)threadIdx.x || slot >= p.cap) odd = 1;
    }
    __syncthreads();
    const bool whole = !odd;
    const uint8_t* heads = p.cache + ((int64_t)b * p.H + h0) * p.cache_blocks * kBlk;
    if (whole) {
        for (int i = threadIdx.x; i < nh * (kBlk / 16); i += 256) {
            const int hi = i / (kBlk / 16), piece = i % (kBlk / 16);
            *reinterpret_cast<u32x4*>(image + hi * kBlk + 16 * piece) = *reinterpret_cast<const u32x4*>(
                heads + (hi * p.cache_blocks + tslot[0] / kKvBlock) * kBlk + 16 * piece);
        }
        __syncthreads();
    }
    const int j = threadIdx.x & (L - 1);
    for (int i = threadIdx.x / L; i < nt * nh * 2; i += kRows) {
        const int sec = i & 1, hi = (i >> 1) % nh, ti = (i >> 1) / nh, slot = tslot[ti];
        float v[8] = {};
        if (slot >= 0 && slot < p.cap) {
            const int tok = slot % kKvBlock;
            if (whole) kv4_get<D>(image + hi * kBlk, tok, sec, j, v);
            else kv4_get<D>(heads + (hi * p.cache_blocks + slot / kKvBlock) * kBlk, tok, sec, j, v);
        }
        store8(p.out[sec], b * p.os[sec][0] + (h0 + hi) * p.os[sec][1] + (s0 + ti) * p.os[sec][2] + 8 * j, p.out_kind, v);
    }
}

static inline int rope_kind(int32_t dt) { return dt == SF_BF16 ? 1 : (dt == SF_F16 ? 2 : 0); }
static inline bool float_dtype(int32_t dt) { return dt == SF_F32 || dt == SF_BF16 || dt == SF_F16; }

// 16-byte aligned rows of D contiguous channels.
static inline bool rows_ok(const void* p, const int64_t st[3]) {
    if (!p || (reinterpret_cast<uintptr_t>(p) & 15)) return false;
    for (int i = 0; i < 3; ++i)
        if (st[i] < 0 || (st[i] & 7)) return false;
    return true;
}

}  // namespace sfk

extern "C" size_t sf_kv4_bytes(int32_t B, int32_t H, int32_t capacity, int32_t D) {
    if (B <= 0 || H <= 0 || capacity <= 0 || (D != 64 && D != 128)) return 0;
    return (size_t)B * (size_t)H * (size_t)sfk::kv4_blocks(capacity) * (size_t)(D * 36);
}

static int kv4_cache_check(const sf_kv4_cache* c) {
    if (!c->data || (reinterpret_cast<uintptr_t>(c->data) & 15) || c->B <= 0 || c->H <= 0 || c->capacity <= 0)
        return SF_EINVAL;
    return c->D == 64 || c->D == 128 ? SF_OK : SF_ENOTSUP;
}

extern "C" int sf_heads_rope(const sf_heads_rope_desc* d, void* stream) {
    if (!d || d->B < 0 || d->S < 0) return SF_EINVAL;
    if (d->D != 64 && d->D != 128) return SF_ENOTSUP;
    if (!sfk::float_dtype(d->in_dtype) || !sfk::float_dtype(d->out_dtype)) return SF_ENOTSUP;
    int64_t heads = 0;
    for (int i = 0; i < 3; ++i) {
        if (d->heads[i] < 0) return SF_EINVAL;
        heads += d->heads[i];
    }
    if (heads == 0 || heads > 65535) return SF_EINVAL;
    if (d->rot < 0 || d->rot > d->D || (d->rot & 15)) return SF_EINVAL;
    if (d->rot && (!d->inv_freq || (reinterpret_cast<uintptr_t>(d->inv_freq) & 7))) return SF_EINVAL;
    const bool cached = d->cache.data != nullptr;
    if (cached) {
        const int st = kv4_cache_check(&d->cache);
        if (st != SF_OK) return st;
        if (d->cache.B != d->B || d->cache.H != d->heads[1] || d->heads[1] != d->heads[2] || d->cache.D != d->D)
            return SF_EINVAL;
    } else if (d->slots) {
        return SF_EINVAL;
    }
    const int64_t tokens = (int64_t)d->B * d->S;
    if (tokens == 0) return SF_OK;
    if (tokens >= 1 << 23) return SF_ENOTSUP;   // a launch counts its threads in 32 bits
    sfk::RopeArgs p = {};
    for (int i = 0; i < 3; ++i) {
        if (!d->heads[i]) continue;
        if (!sfk::rows_ok(d->src[i], d->src_stride[i])) return SF_EINVAL;
        const bool out = i == 0 || !cached;
        if (out && !sfk::rows_ok(d->out[i], d->out_stride[i])) return SF_EINVAL;
        p.src[i] = d->src[i];
        p.out[i] = out ? d->out[i] : nullptr;
        for (int k = 0; k < 3; ++k) p.ss[i][k] = d->src_stride[i][k], p.os[i][k] = d->out_stride[i][k];
    }
    for (int i = 0; i < 2; ++i) {
        if (reinterpret_cast<uintptr_t>(d->gamma[i]) & 3) return SF_EINVAL;
        p.gamma[i] = d->gamma[i];
    }
    p.positions = d->positions;
    p.slots = d->slots;
    p.inv_freq = d->inv_freq;
    p.cache = static_cast<uint8_t*>(d->cache.data);
    p.cache_blocks = cached ? sfk::kv4_blocks(d->cache.capacity) : 0;
    for (int i = 0; i < 3; ++i) p.heads[i] = d->heads[i];
    p.S = d->S;
    p.cap = d->cache.capacity;
    p.rot = d->rot;
    p.interleaved = d->interleaved != 0;
    p.in_kind = sfk::rope_kind(d->in_dtype);
    p.out_kind = sfk::rope_kind(d->out_dtype);
    p.eps = d->eps;
    // Rows to a workgroup.  Into a cache a block's tokens of four heads (4374 tokens x 64 heads: 23.5 us, 26 with
    // eight, 35 with sixteen).  Else four tokens of 32 heads, which share the sines, fewer where there are few tokens:
    // 4374 x 96 heads of 64 channels take 24 us with four, 25.5 with two, 31.5 with eight; 1072 x 96 12.5, 10 and 18.
    const int rows = 256 / (d->D / 8);
    const int spread = tokens >= 2048 ? 4 : tokens >= 512 ? 2 : 1;
    p.tok_per_wg = cached ? (d->S >= sfk::kKvBlock ? sfk::kKvBlock : 1) : spread;
    p.windows = (int)((d->S + (int64_t)p.tok_per_wg - 1) / p.tok_per_wg);
    if (p.tok_per_wg == sfk::kKvBlock && (d->positions || d->slots)) ++p.windows;   // the first one may be cut short
    p.heads_per_wg = (int)std::min<int64_t>(heads, p.tok_per_wg == sfk::kKvBlock ? 4 : p.tok_per_wg > 1 ? 32 : rows);
    p.heads_magic = (65536 + p.heads_per_wg - 1) / p.heads_per_wg;
    const dim3 grid((unsigned)(d->B * p.windows), (unsigned)((heads + p.heads_per_wg - 1) / p.heads_per_wg));
    size_t lds = sizeof(float2) * (size_t)p.tok_per_wg * (size_t)(d->rot / 2);
    if (p.tok_per_wg == sfk::kKvBlock) lds += (size_t)p.heads_per_wg * 18 * d->D;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (d->D == 64) {
        if (cached) hipLaunchKernelGGL((sfk::heads_rope_kernel<64, true>), grid, dim3(256), lds, s, p);
        else hipLaunchKernelGGL((sfk::heads_rope_kernel<64, false>), grid, dim3(256), lds, s, p);
    } else {
        if (cached) hipLaunchKernelGGL((sfk::heads_rope_kernel<128, true>), grid, dim3(256), lds, s, p);
        else hipLaunchKernelGGL((sfk::heads_rope_kernel<128, false>), grid, dim3(256), lds, s, p);
    }
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}

extern "C" int sf_kv4_read(const sf_kv4_cache* cache, const int32_t* slots, int32_t S, void* k, const int64_t* k_stride,
                           void* v, const int64_t* v_stride, int32_t out_dtype, void* stream) {
    if (!cache || S < 0) return SF_EINVAL;
    const int st = kv4_cache_check(cache);
    if (st != SF_OK) return st;
    if (!sfk::float_dtype(out_dtype)) return SF_ENOTSUP;
    if (S == 0) return SF_OK;
    if (!k_stride || !v_stride || !sfk::rows_ok(k, k_stride) || !sfk::rows_ok(v, v_stride)) return SF_EINVAL;
    sfk::Kv4ReadArgs p = {};
    p.cache = static_cast<const uint8_t*>(cache->data);
    p.cache_blocks = sfk::kv4_blocks(cache->capacity);
    p.slots = slots;
    p.out[0] = k;
    p.out[1] = v;
    for (int i = 0; i < 3; ++i) p.os[0][i] = k_stride[i], p.os[1][i] = v_stride[i];
    p.H = cache->H;
    p.S = S;
    p.cap = cache->capacity;
    p.out_kind = sfk::rope_kind(out_dtype);
    if ((int64_t)cache->B * S >= 1 << 23 || cache->H > 65535) return SF_ENOTSUP;   // as sf_heads_rope
    // with slots the first window may be cut short
    p.windows = (int)((S + (int64_t)sfk::kKvBlock - 1) / sfk::kKvBlock) + (slots ? 1 : 0);
    const dim3 grid((unsigned)(cache->B * p.windows), (unsigned)((cache->H + sfk::kReadHeads - 1) / sfk::kReadHeads));
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (cache->D == 64) hipLaunchKernelGGL(sfk::kv4_read_kernel<64>, grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL(sfk::kv4_read_kernel<128>, grid, dim3(256), 0, s, p);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
