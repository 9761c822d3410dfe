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

// Eight channels as loaded.  kind: 0 fp32, 1 bf16, 2 fp16
struct Raw8 {
    u32x4 a, b;   // b: fp32 only
};
__device__ __forceinline__ Raw8 load8(const void* p, int64_t at, int kind) {
    Raw8 r = {};
    if (kind == 0) {
        const u32x4* q = reinterpret_cast<const u32x4*>(static_cast<const float*>(p) + at);
        r.a = q[0];
        r.b = q[1];
    } else {
        r.a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
    }
    return r;
}
__device__ __forceinline__ void widen8(const Raw8& r, int kind, float v[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t u = r.a[e], w = r.b[e];
        if (kind == 0) {
            v[e] = __uint_as_float(u);
            v[4 + e] = __uint_as_float(w);
        } else if (kind == 1) {
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

// Step and middle of a group of 64 channels held by 8 lanes, and the lane's
// eight codes (channel e at nibble e).  The step is a power of two times a
// bf16, so step * integer and x - n * step below carry one rounding at most
// and the code is the floor of the exact quotient, whatever the reciprocal's
// last bit.
__device__ __forceinline__ uint32_t kv4_quantise(const float v[8], uint32_t* par) {
    float mx = v[0], mn = v[0];
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        mx = fmaxf(mx, v[e]);
        mn = fminf(mn, v[e]);
        big = max(big, __float_as_uint(v[e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        mx = fmaxf(mx, __shfl_xor(mx, o, 64));
        mn = fminf(mn, __shfl_xor(mn, o, 64));
        big = max(big, (uint32_t)__shfl_xor((int)big, o, 64));
    }
    if (big >= 0x7f800000u) {   // an infinity or a NaN: the group reads back as NaN
        *par = 0x7fc07fc0u;
        return 0;
    }
    const uint32_t mid_bits = f32_to_bf16_bits(0.5f * mx + 0.5f * mn);
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
        const float d = v[e] - mid;
        float n = floorf(d * inv);
        const float left = __builtin_fmaf(-n, s, d);
        if (left < 0.f) n -= 1.f;
        else if (left >= s) n += 1.f;
        c |= (uint32_t)(int)(fminf(fmaxf(n, -8.f), 7.f) + 8.f) << (4 * e);
    }
    return c;
}

// Nibble e -> nibble (e >> 1) + 4 (e & 1), and back.
__device__ __forceinline__ uint32_t nibbles_to_pairs(uint32_t c) {
    uint32_t o = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) o |= ((c >> (4 * e)) & 15u) << (4 * ((e >> 1) + 4 * (e & 1)));
    return o;
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
    constexpr int L = D / 8, kRows = 256 / L, kAhead = 4;   // rows in flight a thread
    constexpr int kImage = 16 * D + 2 * D;                  // a head's codes and parameters of 32 tokens, keys or values
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    float2* cs = reinterpret_cast<float2*>(lds);                                      // [tok_per_wg][rot / 2]
    uint8_t* image = lds + sizeof(float2) * (size_t)p.tok_per_wg * (p.rot >> 1);      // [heads_per_wg][kImage]
    __shared__ int tpos[kRopeTokens], tslot[kRopeTokens], odd;
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
    for (int base = sub; base - sub < rows; base += kRows * kAhead) {
        Raw8 raw[kAhead];
        int where[kAhead];   // token << 20 | section << 18 | head; -1: none
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int i = base + a * kRows, ti = (i * p.heads_magic) >> 16, hi = i - ti * p.heads_per_wg;
            where[a] = -1;
            if (i >= rows || hi >= nh || tpos[ti] < 0) continue;   // a padding token is not written
            int h = h0 + hi, sec = 0;
            if (h >= p.heads[0]) h -= p.heads[0], sec = 1;
            if (sec == 1 && h >= p.heads[1]) h -= p.heads[1], sec = 2;
            where[a] = ti << 20 | sec << 18 | h;
            raw[a] = load8(p.src[sec], b * p.ss[sec][0] + h * p.ss[sec][1] + (s0 + ti) * p.ss[sec][2] + 8 * j, p.in_kind);
        }
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            if (where[a] < 0) continue;   // whole groups of L lanes
            const int ti = where[a] >> 20, sec = where[a] >> 18 & 3, h = where[a] & 0x3ffff;
            float v[8];
            widen8(raw[a], p.in_kind, v);
            const float* gm = sec == 0 ? p.gamma[0] : sec == 1 ? p.gamma[1] : nullptr;
            if (gm) {
                float q = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) q += v[e] * v[e];
                q = L == 8 ? row8_sum(q) : row16_sum(q);
                const float r = 1.f / sqrtf(q / (float)D + p.eps);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = v[e] * r * gm[8 * j + e];
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
                // where the block's codes and parameters lie: in the cache, or in this head's image
                const int tok = slot % kKvBlock, head = (int)(sec == 1 ? p.heads[0] + h : p.heads[0] + p.heads[1] + h) - h0;
                uint8_t* blk = whole ? image + head * kImage
                                     : p.cache + (((int64_t)b * p.heads[1] + h) * p.cache_blocks + slot / kKvBlock) * Kv4<D>::kBytes;
                uint8_t* pars = blk + (whole ? 16 * D : sec == 1 ? Kv4<D>::kPar : Kv4<D>::kVPar);
                if ((j & 7) == 0) *reinterpret_cast<uint32_t*>(pars + ((j >> 3) * kKvBlock + tok) * 4) = par;
                if (sec == 1) {
                    *reinterpret_cast<uint32_t*>(blk + Kv4<D>::key_dword(tok, j)) = nibbles_to_pairs(c);
                } else {
                    // lanes j and j ^ 2 hold channels 16 apart: each writes four of the eight bytes they share
                    const bool hi = j & 2;
                    const uint32_t lo = hi ? other : c, up = hi ? c : other;
                    const int first = hi ? 4 : 0, at = whole ? Kv4<D>::kV : 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int sh = 4 * (first + e);
                        blk[Kv4<D>::value_byte(tok, j >> 2, 8 * (j & 1) + first + e) - at] =
                            (uint8_t)(((lo >> sh) & 15u) | ((up >> sh) & 15u) << 4);
                    }
                }
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

struct Kv4ReadArgs {
    const uint8_t* cache;
    int64_t cache_blocks;
    const int32_t* slots;
    void* out[2];
    int64_t os[2][3];
    int H, S, cap, out_kind;
    int64_t rows;   // B * S * H * 2
};

// The values of given slots: one row of D / 8 lanes per (token, head, K or V).
template <int D>
__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4ReadArgs p) {
    constexpr int L = D / 8, kRows = 256 / L;
    const int j = threadIdx.x & (L - 1);
    const int64_t i = (int64_t)blockIdx.x * kRows + threadIdx.x / L;
    if (i >= p.rows) return;
    const int sec = (int)(i & 1), h = (int)((i >> 1) % p.H);
    const int64_t m = (i >> 1) / p.H, b = m / p.S;
    const int s = (int)(m % p.S);
    const int slot = p.slots ? p.slots[m] : s;
    float v[8];
    if (slot < 0 || slot >= p.cap) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
    } else {
        const uint8_t* blk = p.cache + ((b * p.H + h) * p.cache_blocks + slot / kKvBlock) * Kv4<D>::kBytes;
        const int tok = slot % kKvBlock;
        const uint32_t par = *reinterpret_cast<const uint32_t*>(
            blk + (sec ? Kv4<D>::value_par(tok, j >> 3) : Kv4<D>::key_par(tok, j >> 3)));
        const float st = __uint_as_float(par << 16), mid = __uint_as_float(par & 0xffff0000u);
        const uint32_t c = sec ? 0u : *reinterpret_cast<const uint32_t*>(blk + Kv4<D>::key_dword(tok, j));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            uint32_t n = (c >> (4 * ((e >> 1) + 4 * (e & 1)))) & 15u;
            if (sec) n = ((uint32_t)blk[Kv4<D>::value_byte(tok, j >> 2, 8 * (j & 1) + e)] >> (j & 2 ? 4 : 0)) & 15u;
            v[e] = __builtin_fmaf((float)n - 7.5f, st, mid);
        }
    }
    store8(p.out[sec], b * p.os[sec][0] + h * p.os[sec][1] + s * p.os[sec][2] + 8 * j, p.out_kind, v);
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
    if (tokens > 0x7fffffffLL) return SF_ENOTSUP;
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
    // A few hundred rows to a workgroup where there are many, one pass of its threads where there are few.
    const int rows = 256 / (d->D / 8);
    const bool many = tokens >= 512;
    p.tok_per_wg = cached ? (d->S >= sfk::kKvBlock ? sfk::kKvBlock : 1) : many ? 8 : 1;
    p.windows = (int)((d->S + (int64_t)p.tok_per_wg - 1) / p.tok_per_wg);
    if (p.tok_per_wg == sfk::kKvBlock && (d->positions || d->slots)) ++p.windows;   // the first one may be cut short
    p.heads_per_wg = (int)std::min<int64_t>(heads, p.tok_per_wg == sfk::kKvBlock ? 8 : many ? 32 : rows);
    p.heads_magic = (65536 + p.heads_per_wg - 1) / p.heads_per_wg;
    const int64_t wgs = (int64_t)d->B * p.windows;
    if (wgs > 0x7fffffffLL) return SF_ENOTSUP;
    const dim3 grid((unsigned)wgs, (unsigned)((heads + p.heads_per_wg - 1) / p.heads_per_wg));
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
    p.rows = (int64_t)cache->B * S * cache->H * 2;
    const int rows = 256 / (cache->D / 8);
    const int64_t blocks = (p.rows + rows - 1) / rows;
    if ((int64_t)cache->B * S > 0x7fffffffLL || blocks > 0x7fffffffLL) return SF_ENOTSUP;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (cache->D == 64) hipLaunchKernelGGL(sfk::kv4_read_kernel<64>, dim3((unsigned)blocks), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(sfk::kv4_read_kernel<128>, dim3((unsigned)blocks), dim3(256), 0, s, p);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
