// Attention over the 4-bit key / value cache (gfx950).
//
// A cached value is s (c - 7.5) + mid with s and mid of its token, head and
// 64-channel group, so both contractions run on the codes themselves and the
// parameters meet the scores in fp32:
//   S_j = s_j sum_d q_d (16 + c_jd) + (mid_j - 23.5 s_j) sum_d q_d
//   O_d = sum_j p_j s_j (16 + c_jd) - 23.5 sum_j p_j s_j + sum_j p_j mid_j
// (16 + c: see sf_nibble.h).  p_j s_j enters the matrix unit as a bf16 (hi, lo)
// pair, 2^-18 relative, and its sum is taken over the same rounded pair, so that
// what the codes' offset adds is taken away exactly; for fp32 outputs it enters as
// three terms.  With many query rows that see the same tokens and a bf16 output the
// values are formed in fp16 instead, once for all rows, and p enters as one fp16:
// five vector operations fewer for every score, and roundings of 2^-11 where the
// output's own is 2^-8 (6e-4 of its norm beside 1.7e-3); exact_pv keeps the pair.
//
// One wave takes blocks of 32 tokens against QT tiles of 16 query rows; query
// heads that share a key head are rows of one tile, so a cached token is read
// and unpacked once for all of them.  S^T = K Q^T puts a row's scores in the
// lanes that the second product wants them in as P^T (the cache's value order,
// sf_kv4.h): no score passes through LDS.  What does, inside the loop, are the
// queries of more than one tile, read back as operands, and with them the raw
// blocks of 128 channels.  The running maximum moves only when a score exceeds it
// by 2^8: p stays below 2^8, far inside bf16 and fp32, and the common block has
// neither a cross-lane maximum nor a rescale.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "sf_device.h"
#include "sf_hip.h"
#include "sf_kv4.h"
#include "sf_nibble.h"

namespace sfk {

constexpr int kKvMaxSplits = 64;
constexpr float kKvSlack = 8.f;       // log2
constexpr int64_t kKvMergeRows = 1 << 24;   // the merge's workgroups: a launch counts its threads in 32 bits
constexpr int kKvHalfKeys = 4096;     // of a wave, with weights in fp16
constexpr float kKvNoMax = -1.5e38f;  // the maximum of a row that has seen nothing

// How p and V meet.  kKvHalf (bf16 outputs of many rows that see the same tokens):
// both in fp16.  Not for causal rows: what later rows alone see would set the power
// under which an earlier row's values are rounded, and a NaN among it, as V, would
// reach rows whose weight for it is 0.  Nor for more than 4096 keys of a wave: a
// weight below 2^-14 of the wave's largest is held to 2^-25 only, one below 2^-25
// not at all, which N keys make N 2^-24 of the largest value (2^-12 for 4096).
// (Causal, us with the pair, and with fp16 when the blocks that some rows see a part
// of are taken in steps of values of like size: 64 channels, 8 heads of 4 x 256 rows
// over 2048 keys, twice, 18.5 and 17.5, of 4 x 4096 over 4096 193 and 168; 128
// channels, the first of these 30.5 and 34.8.)  kKvPair (other 16-bit outputs): p s
// as a bf16 (hi, lo) pair with the codes, whose offset the pairs' sums take away at
// the end.  kKvExact (fp32 outputs): three terms instead of two, and the offset,
// which is many times a mean of values and would leave its own rounding, is taken
// away inside the products: -23.5 times the queries' sums under the scores, a
// product with -23.5 beside each block's.  Of the output's norm that is off by
// 1.3e-7 (20 keys) to 7e-7 (8192), as the same sums over fp32 values are, where the
// pair is off by 1.4e-6 to 1e-5; it costs 16 x 8 heads x 16384 keys x 4 rows 78 us
// instead of 70, 4 x 32 x 4374 x 67 rows 48 instead of 40, and 4 x 8 x 4096 x 268
// rows of 128 channels, which spill, 110 instead of 87.
enum { kKvHalf, kKvPair, kKvExact };

struct KvAttnArgs {
    const uint16_t* q;
    const uint8_t* cache;
    void* out;
    float* part;          // [splits][rows][D + 2], rows = B * Hq * Sq: O, then max and sum
    const int32_t* valid;
    const uint8_t* mask;
    int64_t mask_stride, cache_blocks;
    int64_t qs[3], os[3];
    int64_t rows;
    int B, H, G, Sq, Sk, splits, qgroups, causal, out_kind;
    float scale_log2;
    const uint32_t* tree;   // [B or 1][T][words]: bit i of a node's row is set where it sees node i
    int64_t tree_stride;    // words between batch elements, 0 for one tree
    int T, tree_words;
};

// A tree: the T nodes are the last T tokens, all before them are seen by every row.  Which of
// the 32 tokens from key0 on the row of node `node` sees, the nodes' first token at key `at`:
// two words of its ancestors, shifted.  Only the T / 32 + 1 blocks that hold nodes ask; all before
// them run as a call without a tree, so the rows cost what they cost there.  us: 16 x 8 heads x 64
// rows (16 nodes) over 2048..8192 keys of 128 channels 79, of a floor of 19: the pair's vector
// work, done for two groups of 32 rows that each unpack the block, and the longest sequence, whose
// workgroups have a CU each (in equal pieces of 4096, 2048, 1024 keys 96, 98 and 115, beside 83: a workgroup's
// start, join and merge cost more than the balance gains); 4 x 32 heads x 64 rows over 1094..4374
// keys of 64 29, of 5.
__device__ __forceinline__ uint32_t kv_tree_bits(const KvAttnArgs& p, int b, int node, int key0, int at) {
    const uint32_t* row = p.tree + b * p.tree_stride + (int64_t)node * p.tree_words;
    const int r = key0 - at, w = r >> 5;   // rounded down
    const uint32_t lo = w < 0 ? ~0u : w < p.tree_words ? row[w] : 0u;
    const uint32_t hi = w + 1 < 0 ? ~0u : w + 1 < p.tree_words ? row[w + 1] : 0u;
    return (uint32_t)(((uint64_t)hi << 32 | lo) >> (r & 31));
}

// A lane's 8 tokens of a block's 32 bits: 4 g .. + 3 and 16 + 4 g .. + 3.
__device__ __forceinline__ uint32_t kv_lane_bits(uint32_t bits, int g) {
    return (bits >> (4 * g) & 15u) | (bits >> (16 + 4 * g) & 15u) << 4;
}

// N consecutive channels to out: kind 0 fp32, 1 bf16, 2 fp16 (stores of 2 N and 4 N bytes, N even).
template <int N>
__device__ __forceinline__ void kv_store(void* out, int64_t at, int kind, const float (&y)[N]) {
    typedef float fv __attribute__((ext_vector_type(N)));
    typedef uint32_t uv __attribute__((ext_vector_type(N / 2)));
    if (kind == 0) {
        fv v;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = y[e];
        *reinterpret_cast<fv*>(static_cast<float*>(out) + at) = v;
        return;
    }
    uv u;
#pragma unroll
    for (int e = 0; e < N / 2; ++e)
        u[e] = kind == 1 ? pack_bf16x2(y[2 * e], y[2 * e + 1]) : pack_f16x2_rn(y[2 * e], y[2 * e + 1]);
    *reinterpret_cast<uv*>(static_cast<uint16_t*>(out) + at) = u;
}

__device__ __forceinline__ float lanes4_sum(float x) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}
__device__ __forceinline__ float lanes4_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}

// a s + b mid of a parameter dword, in fp32; a and b are bf16 numbers.
__device__ __forceinline__ float kv_mix(uint32_t par, float a, float b) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, par), bf16x2v{(__bf16)a, (__bf16)b}, 0.f, false);
}

// acc - 23.5 times the sum of a pair of bf16.
__device__ __forceinline__ float kv_dot(uint32_t pair, float acc) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, pair), bf16x2v{(__bf16)-23.5f, (__bf16)-23.5f}, acc, false);
}

// The exponent, offset by 127 as in fp32, of the larger of 2^18 s and |mid| of a parameter dword (0: a NaN, or nothing
// above the subnormals).
__device__ __forceinline__ uint32_t kv_size(uint32_t par) {
    const uint32_t s = par >> 7 & 0xffu, mid = par >> 23 & 0xffu;
    return s == 0xffu ? 0u : max(s ? s + 18u : 0u, mid);
}

// A matrix operand of -23.5.
__device__ __forceinline__ u32x4 kv_offset() { return u32x4{0xC1BCC1BCu, 0xC1BCC1BCu, 0xC1BCC1BCu, 0xC1BCC1BCu}; }

// What a wave holds of a block of 32 tokens.
template <int D>
struct KvBlock {
    static constexpr int G = D / 64;
    u32x4 k[G], v[G];                       // codes
    u32x4 kp[G][2], vp[G][2];               // parameters of tokens 4 g .. + 3 and 16 + 4 g .. + 3
    __device__ __forceinline__ void load(const uint8_t* blk, int lane) {
        const int g = lane >> 4;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            k[i] = *reinterpret_cast<const u32x4*>(blk + i * 1024 + lane * 16);
            v[i] = *reinterpret_cast<const u32x4*>(blk + Kv4<D>::kV + i * 1024 + lane * 16);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                kp[i][t] = *reinterpret_cast<const u32x4*>(blk + Kv4<D>::key_par(16 * t + 4 * g, i));
                vp[i][t] = *reinterpret_cast<const u32x4*>(blk + Kv4<D>::value_par(16 * t + 4 * g, i));
            }
        }
    }
    // Key code dword of tile t, group i, step ks.
    __device__ __forceinline__ uint32_t key(int t, int i, int ks) const {
        return D == 64 ? k[0][2 * t + ks] : k[t][2 * i + ks];
    }
};

// The rare step of the running maximum: a row's scores x (less the old maximum
// m, or as they are in a row that has seen nothing) exceed it by the slack.
// Returns what the row's sums are to be scaled by.
__device__ __forceinline__ float kv_raise(float (&x)[8], float mx, float& m) {
    const bool first = m == kKvNoMax;
    const float top = lanes4_max(mx), up = first ? (top == -INFINITY ? 0.f : top) : fmaxf(0.f, top);
    m = first ? (top == -INFINITY ? kKvNoMax : top) : m + up;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] -= up;
    return first ? 1.f : __builtin_amdgcn_exp2f(-up);   // first: nothing to scale
}

// A query row's operand (channels 64 i + 16 g .. + 15 of the lane's group g) and
// the sums of its channels.
template <bool F16, int D>
__device__ __forceinline__ void kv_queries(const KvAttnArgs& p, int b, int hq, int s, int g, u32x4 (&f)[D / 64][2],
                                           float (&sums)[D / 64]) {
    const uint16_t* src = p.q + b * p.qs[0] + hq * p.qs[1] + s * p.qs[2];
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) f[i][k] = *reinterpret_cast<const u32x4*>(src + 64 * i + 16 * g + 8 * k);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t v = f[i][k][e];
                sum += F16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)v) + (float)__builtin_bit_cast(_Float16, (uint16_t)(v >> 16))
                           : __uint_as_float(v << 16) + __uint_as_float(v & 0xffff0000u);
            }
        sums[i] = lanes4_sum(sum);
    }
}

// A joined row: its output, or its sums for the merge of key splits.
template <int D, int E>
__device__ __forceinline__ void kv_finish(const KvAttnArgs& p, int split, int b, int hq, int s, int d0, float (&y)[E],
                                          float top, float sum) {
    if (p.splits > 1) {
        float* dst = p.part + ((int64_t)split * p.rows + ((int64_t)b * p.H * p.G + hq) * p.Sq + s) * (D + 2);
#pragma unroll
        for (int e = 0; e < E; ++e) dst[d0 + e] = y[e];
        if (d0 == 0) dst[D] = top, dst[D + 1] = sum;
    } else {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;   // nothing visible: zeros
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] *= inv;
        kv_store<E>(p.out, b * p.os[0] + hq * p.os[1] + s * p.os[2] + d0, p.out_kind, y);
    }
}

// QT tiles of 16 query rows of a key head to a workgroup.
template <bool F16, int D, int QT, int FORM, int NW, bool TREE = false>
__global__ __launch_bounds__(64 * NW) void attn_kv4_kernel(const KvAttnArgs p) {
    constexpr int GR = D / 64, DT = D / 16;   // 64-channel groups, tiles of 16 channels
    constexpr bool PAIR = FORM != kKvHalf, EXACT = FORM == kKvExact;
    static_assert(PAIR || !TREE, "rows of a tree see different tokens");
    __shared__ float xm[NW][QT * 16], xl[NW][QT * 16], xf[NW][QT * 16], xs[QT * 16];
    constexpr int kJoin = D == 128 && NW == 8 ? 1 : QT == 5 ? 3 : QT == 4 ? 2 : QT;   // tiles that meet at a time
    // 128 channels and two tiles leave no registers for the next raw block beside eight waves: it waits in LDS, brought
    // there straight from memory.  us, against four waves with it in registers: 8 x 32 heads x 67 x 4374 145 and 166,
    // 2 x 8 x 268 rows x 8192 73 and 96 (129 and 70 since the fp16 form knows no causal rows and does not spill).
    constexpr bool kStaged = D == 128 && QT > 1;
    __shared__ __attribute__((aligned(16))) uint8_t raw[kStaged ? NW : 1][kStaged ? Kv4<D>::kBytes : 16];
    __shared__ float xo[NW][kJoin * 16][D + 4], xq[GR][QT * 16];
    __shared__ u32x4 ql[QT > 1 ? QT * GR * 2 : 1][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, g = lane >> 4;
    const int split = blockIdx.x % p.splits;
    const int qg = (blockIdx.x / p.splits) % p.qgroups;
    const int bh = blockIdx.x / p.splits / p.qgroups;
    const int b = bh / p.H, h = bh % p.H;
    const int R = p.G * p.Sq, q0 = qg * 16 * QT;

    const int len = p.valid ? min(max(p.valid[b], 0), p.Sk) : p.Sk;
    // Query s sees keys below len - Sq + s + 1 (causal) or len; the smallest and largest limit of the group's rows.
    int lim_lo = TREE ? len - p.T : len, lim_hi = len;
    if (PAIR && !TREE && p.causal) {
        const int q1 = min(q0 + 16 * QT, R) - 1;
        const bool one = q0 / p.Sq == q1 / p.Sq;
        lim_lo = len - p.Sq + 1 + (one ? q0 % p.Sq : 0);
        lim_hi = len - p.Sq + 1 + (one ? q1 % p.Sq : p.Sq - 1);
    }
    const int nblk = (max(lim_hi, 0) + kKvBlock - 1) / kKvBlock;
    const int b0 = (int)((int64_t)nblk * split / p.splits), b1 = (int)((int64_t)nblk * (split + 1) / p.splits);

    const uint8_t* base = p.cache + (int64_t)bh * p.cache_blocks * Kv4<D>::kBytes;
    KvBlock<D> nx;
    auto fetch = [&](int blk) __attribute__((always_inline)) {
        const uint8_t* from = base + (int64_t)(kStaged ? __builtin_amdgcn_readfirstlane(blk) : blk) * Kv4<D>::kBytes;
        if constexpr (kStaged) {
            const __amdgpu_buffer_rsrc_t blocks = make_rsrc(from, Kv4<D>::kBytes);
            const int w = __builtin_amdgcn_readfirstlane(wave);
            int at_lane = 16 * lane;
            asm volatile("" : "+v"(at_lane));   // or 4 * lane is kept in a register, which spills
#pragma unroll
            for (int at = 0; at < 32 * D; at += 1024)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(blocks, (__attribute__((address_space(3))) void*)(raw[w] + at), 16,
                                                         at_lane, at, 0, 0);
#pragma unroll
            for (int at = 32 * D; at < 36 * D; at += 256)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(blocks, (__attribute__((address_space(3))) void*)(raw[w] + at), 4,
                                                         at_lane >> 2, at, 0, 0);
        } else {
            nx.load(from, lane);
        }
    };
    if (b0 + wave < b1) fetch(b0 + wave);

    // Query fragments (B operands) and row sums: in registers for one tile, else each tile's by one wave into LDS.
    static_assert(QT <= NW, "a wave for each tile");
    u32x4 qr[GR][2];
    float qs[QT][GR], off[QT][GR];   // scale * log2 e times a row's sum; what the codes' offset adds to its scores
    if (QT == 1 || wave < QT) {
        const int t = QT == 1 ? 0 : wave, r = min(q0 + 16 * t + col, R - 1);
        kv_queries<F16, D>(p, b, h * p.G + r / p.Sq, r % p.Sq, g, qr, qs[0]);
        if (QT > 1) {
#pragma unroll
            for (int i = 0; i < GR; ++i) {
                ql[(t * GR + i) * 2][lane] = qr[i][0];
                ql[(t * GR + i) * 2 + 1][lane] = qr[i][1];
                if (g == 0) xq[i][16 * t + col] = qs[0][i];
            }
        }
    }
    if (QT > 1) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
            for (int i = 0; i < GR; ++i) qs[t][i] = xq[i][16 * t + col];
    }
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            off[t][i] = EXACT ? -23.5f * qs[t][i] : 0.f;
            qs[t][i] *= p.scale_log2;
        }

    f32x4 o[QT][DT];   // O^T; PAIR: without the parameters' part pm
    float m[QT], l[QT], pm[QT][PAIR ? GR : 1];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        m[t] = kKvNoMax, l[t] = 0.f;
#pragma unroll
        for (int i = 0; i < (PAIR ? GR : 1); ++i) pm[t][i] = 0.f;
#pragma unroll
        for (int i = 0; i < DT; ++i) o[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // fp16 form: values are held times `vdown`, a power of two of the wave's that keeps 2^18 s and |mid - 7.5 s| of
    // every token seen below 2^15; the first block sets it, a larger one lowers it.
    float vdown = 1.f / 262144.f, vcap = 0.f;
    const NibbleMask kmask = nibble_mask<F16>(), vmask = nibble_mask<false>();

    auto block = [&](const int blk, auto masked_c) __attribute__((always_inline)) {
        constexpr bool masked = decltype(masked_c)::value;
        const int key0 = kKvBlock * blk;
        if (kStaged) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            nx.load(raw[kStaged ? wave : 0], lane);
        }
        uint32_t see = 0xffu;   // the lane's 8 tokens, by length and mask
        if (masked) {
            see = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = key0 + 16 * (e >> 2) + 4 * g + (e & 3);
                if (key < len && (!p.mask || p.mask[b * p.mask_stride + key])) see |= 1u << e;
            }
        }
        uint32_t mine[TREE && masked ? QT : 1];   // the lane's tokens, by each tile's rows
        if constexpr (TREE && masked) {
#pragma unroll
            for (int t = 0; t < QT; ++t)
                mine[t] = kv_lane_bits(kv_tree_bits(p, b, p.T - p.Sq + min(q0 + 16 * t + col, R - 1) % p.Sq, key0, len - p.T), g);
        }
        float ks[GR][8], ko[GR][8], vs[GR][8], vm[GR][8];
#pragma unroll
        for (int i = 0; i < GR; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint32_t kp = nx.kp[i][e >> 2][e & 3], vp = nx.vp[i][e >> 2][e & 3];
                if (masked && !(see >> e & 1u)) kp = vp = 0u;   // tokens behind the last hold anything
                ks[i][e] = __uint_as_float(kp << 16) * p.scale_log2;
                ko[i][e] = EXACT ? __uint_as_float(kp & 0xffff0000u) : kv_mix(kp, -23.5f, 1.f);
                vs[i][e] = PAIR ? __uint_as_float(vp << 16) : kv_mix(vp, 262144.f * vdown, 0.f);
                vm[i][e] = PAIR ? __uint_as_float(vp & 0xffff0000u) : kv_mix(vp, -7.5f * vdown, vdown);
            }
        u32x4 ka[2][GR][2], va[DT];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < GR; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) ka[t][i][k] = nibbles_plus16<F16>(nx.key(t, i, k), kmask);
        if (!PAIR) {
            float big = 0.f;
#pragma unroll
            for (int i = 0; i < GR; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) big = fmaxf(fmaxf(big, vs[i][e]), fabsf(vm[i][e]));
            if (__any(big > vcap)) {   // a new power: this block's largest to 2^12 .. 2^13
                // From the parameters themselves: times the old power they may have passed fp32's range.
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < GR; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (!masked || (see >> e & 1u)) top = max(top, kv_size(nx.vp[i][e >> 2][e & 3]));
#pragma unroll
                for (int w = 16; w < 64; w <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, w, 64));   // a group's 16 lanes hold the same
                const int now = (int)(__float_as_uint(vdown) >> 23) - 127;
                const int ex = __builtin_amdgcn_readfirstlane(min(max(127 + 12 - (int)top, -126), 100));
                const float al = __builtin_amdgcn_ldexpf(1.f, ex - now);
                vdown = __uint_as_float((uint32_t)(127 + ex) << 23);
                vcap = 32768.f;
#pragma unroll
                for (int t = 0; t < QT; ++t)
#pragma unroll
                    for (int i = 0; i < DT; ++i) o[t][i] *= al;
#pragma unroll
                for (int i = 0; i < GR; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint32_t vp = nx.vp[i][e >> 2][e & 3];
                        if (masked && !(see >> e & 1u)) vp = 0u;
                        vs[i][e] = kv_mix(vp, 262144.f * vdown, 0.f);
                        vm[i][e] = kv_mix(vp, -7.5f * vdown, vdown);
                    }
            }
        }
#pragma unroll
        for (int t = 0; t < DT / 2; ++t) {
            const uint32_t w0 = nx.v[t >> 1][2 * (t & 1)], w1 = nx.v[t >> 1][2 * (t & 1) + 1];
            if (PAIR) {
                va[2 * t] = u32x4{nibble_pair_plus16<false, 0>(w0, vmask), nibble_pair_plus16<false, 2>(w0, vmask),
                                  nibble_pair_plus16<false, 0>(w1, vmask), nibble_pair_plus16<false, 2>(w1, vmask)};
                va[2 * t + 1] = u32x4{nibble_pair_plus16<false, 1>(w0, vmask), nibble_pair_plus16<false, 3>(w0, vmask),
                                      nibble_pair_plus16<false, 1>(w1, vmask), nibble_pair_plus16<false, 3>(w1, vmask)};
            } else {   // c 2^-18 as fp16 subnormals, then pairs of tokens' c s + (mid - 7.5 s) with one rounding
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = e < 2 ? w0 : w1;
                    const uint32_t lo = e & 1 ? w >> 2 : w << 6, hi = e & 1 ? w >> 6 : w << 2;
                    const f16x2v sp = __builtin_bit_cast(f16x2v, pack_f16x2_rn(vs[t >> 1][2 * e], vs[t >> 1][2 * e + 1]));
                    const f16x2v mp = __builtin_bit_cast(f16x2v, pack_f16x2_rn(vm[t >> 1][2 * e], vm[t >> 1][2 * e + 1]));
                    va[2 * t][e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2v, lo & 0x03C003C0u), sp, mp));
                    va[2 * t + 1][e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(f16x2v, hi & 0x03C003C0u), sp, mp));
                }
            }
        }
        // the raw block is spent: fetch the wave's next one
        if (kStaged) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next one comes into its place
        if (blk + NW < b1) fetch(blk + NW);

        // Raw scores of a tile; the next one's products are issued before this one's exponentials, its operands
        // read before this one's maximum.
        f32x4 s[2][GR];
        u32x4 qf[GR][2];
        auto operands = [&](int t) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < GR; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) qf[i][k] = QT == 1 ? qr[i][k] : ql[(t * GR + i) * 2 + k][lane];
        };
        auto scores = [&](int t) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < GR; ++i)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                    s[kt][i] = mfma_16b<F16>(ka[kt][i][1], qf[i][1], mfma_16b<F16>(ka[kt][i][0], qf[i][0], f32x4{off[t][i], off[t][i], off[t][i], off[t][i]}));
        };
        operands(0);
        scores(0);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            if (t + 1 < QT) operands(t + 1);
            float x[8];   // scores less the row's maximum, base 2
            const float neg = m[t] == kKvNoMax ? 0.f : -m[t];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float u = neg;
#pragma unroll
                    for (int i = 0; i < GR; ++i)
                        u = __builtin_fmaf(ks[i][4 * kt + e], s[kt][i][e], __builtin_fmaf(ko[i][4 * kt + e], qs[t][i], u));
                    x[4 * kt + e] = u;
                }
            uint32_t row = see;
            if constexpr (TREE && masked) {
                row &= mine[t];
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(row >> e & 1u)) x[e] = -INFINITY;
            } else if (masked) {
                const int limit = PAIR && p.causal ? len - p.Sq + 1 + min(q0 + 16 * t + col, R - 1) % p.Sq : len;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (key0 + 16 * (e >> 2) + 4 * g + (e & 3) >= limit) row &= ~(1u << e);
                    if (!(row >> e & 1u)) x[e] = -INFINITY;
                }
            }
            const float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            if (__any(mx > (m[t] == kKvNoMax ? -INFINITY : kKvSlack))) {
                const float al = kv_raise(x, mx, m[t]);
                l[t] *= al;
#pragma unroll
                for (int i = 0; i < (PAIR ? GR : 1); ++i) pm[t][i] *= al;
#pragma unroll
                for (int i = 0; i < DT; ++i) o[t][i] *= al;
            }
            if (t + 1 < QT) scores(t + 1);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __builtin_amdgcn_exp2f(x[e]);
            if (PAIR) {
#pragma unroll
                for (int e = 0; e < 8; ++e) l[t] += x[e];
#pragma unroll
                for (int i = 0; i < GR; ++i) {
                    u32x4 hi, lo, rest;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float a = x[2 * e] * vs[i][2 * e], c = x[2 * e + 1] * vs[i][2 * e + 1];
                        float ma = x[2 * e] * vm[i][2 * e], mc = x[2 * e + 1] * vm[i][2 * e + 1];
                        if (masked) {   // a token that only later rows see may hold NaN parameters
                            if (!(row >> (2 * e) & 1u)) a = ma = 0.f;
                            if (!(row >> (2 * e + 1) & 1u)) c = mc = 0.f;
                        }
                        const uint32_t h = pack_bf16x2(a, c);
                        a -= __uint_as_float(h << 16), c -= __uint_as_float(h & 0xffff0000u);
                        const uint32_t w = pack_bf16x2(a, c);
                        pm[t][i] = EXACT ? pm[t][i] + ma + mc : kv_dot(h, kv_dot(w, pm[t][i] + ma + mc));
                        hi[e] = h;
                        lo[e] = w;
                        if (EXACT) rest[e] = pack_bf16x2(a - __uint_as_float(w << 16), c - __uint_as_float(w & 0xffff0000u));
                    }
#pragma unroll
                    for (int d = 4 * i; d < 4 * i + 4; ++d) {
                        if (EXACT) o[t][d] = mfma_16b<false>(kv_offset(), hi, o[t][d]);
                        o[t][d] = mfma_16b<false>(va[d], lo, mfma_16b<false>(va[d], hi, o[t][d]));
                        if (EXACT) {   // the small terms where the sum is small again
                            o[t][d] = mfma_16b<false>(va[d], rest, mfma_16b<false>(kv_offset(), lo, o[t][d]));
                            o[t][d] = mfma_16b<false>(kv_offset(), rest, o[t][d]);
                        }
                    }
                }
            } else {   // the sum is taken over the rounded p, as the product is
                u32x4 ph;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = pack_f16x2_rn(x[2 * e], x[2 * e + 1]);
                    ph[e] = w;
                    l[t] = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2v, w), f16x2v{(_Float16)1.f, (_Float16)1.f}, l[t], false);
                }
#pragma unroll
                for (int d = 0; d < DT; ++d) o[t][d] = mfma_16b<true>(va[d], ph, o[t][d]);
            }
        }
    };
    // Two waves of a workgroup share a SIMD, and the older one wins every tie: it would end first and leave the other
    // to run alone.  A wave's priority falls as it gets on, so the one behind goes first.
    int pace = 3;
    __builtin_amdgcn_s_setprio(3);
    for (int blk = b0 + wave; blk < b1; blk += NW) {
        const int left = b1 - __builtin_amdgcn_readfirstlane(blk), all = b1 - b0;   // priority 3 for 40% of the way, 2 to 70%, 1 to 90%
        const int now = 10 * left > 6 * all ? 3 : 10 * left > 3 * all ? 2 : 10 * left > all ? 1 : 0;
        if (now != pace) {
            if (now == 2) __builtin_amdgcn_s_setprio(2);
            else if (now == 1) __builtin_amdgcn_s_setprio(1);
            else __builtin_amdgcn_s_setprio(0);
            pace = now;
        }
        if (p.mask || kKvBlock * (blk + 1) > lim_lo) block(blk, std::true_type{});
        else block(blk, std::false_type{});
    }

    // The waves' rows meet: what each wave's sums count of a row, then tile by tile through LDS, every thread a
    // piece of a row.
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        l[t] = lanes4_sum(l[t]);
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            const float add = PAIR ? lanes4_sum(pm[t][PAIR ? i : 0]) : 0.f;
#pragma unroll
            for (int d = 4 * i; d < 4 * i + 4; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[t][d][e] += add;
        }
        if (g == 0) xm[wave][16 * t + col] = m[t], xl[wave][16 * t + col] = l[t];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < QT * 16; i += 64 * NW) {
        float mm = xm[0][i], sum = 0.f;
#pragma unroll
        for (int w = 1; w < NW; ++w) mm = fmaxf(mm, xm[w][i]);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(xm[w][i] - mm);
            xf[w][i] = f;
            sum += f * xl[w][i];
        }
        xs[i] = sum;
        xm[0][i] = mm;   // this thread's alone
    }
    __syncthreads();
    constexpr int E = D / (4 * NW);   // channels a thread finishes of a row of each tile
    const int row = (int)threadIdx.x / (4 * NW), d0 = E * ((int)threadIdx.x % (4 * NW));
    const float undo = PAIR ? 1.f : 1.f / vdown;
#pragma unroll
    for (int t0 = 0; t0 < QT; t0 += kJoin) {
        if (t0) __syncthreads();
#pragma unroll
        for (int j = 0; j < kJoin; ++j) {
            if (t0 + j >= QT) continue;
            const float f = xf[wave][16 * (t0 + j) + col] * undo;
#pragma unroll
            for (int d = 0; d < DT; ++d)
                *reinterpret_cast<f32x4*>(&xo[wave][16 * j + col][16 * d + 4 * g]) = o[t0 + j][d] * f;
        }
        __syncthreads();
        for (int j = 0; j < kJoin && t0 + j < QT; ++j) {
            const int r = q0 + 16 * (t0 + j) + row;
            if (r >= R) break;
            float y[E];
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = xo[0][16 * j + row][d0 + e];
#pragma unroll
            for (int w = 1; w < NW; ++w)
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] += xo[w][16 * j + row][d0 + e];
            kv_finish<D, E>(p, split, b, h * p.G + r / p.Sq, r % p.Sq, d0, y, xm[0][16 * (t0 + j) + row], xs[16 * (t0 + j) + row]);
        }
    }
}

// Up to 16 / NG query rows to a key head: one token's heads, or a few tokens'.
//
// One tile of 16 columns would repeat its rows NG times over.  Instead column
// group j of the tile takes block j of the wave's NG blocks at a time: all NG
// blocks' codes meet the tile, each with the queries only in its own columns, so
// the scores of a group's columns are its block's alone, and everything that is
// done per score -- the parameters, the exponentials, the rounded weights -- is
// done once for NG blocks.  The column groups are joined at the end like waves.
// 128 channels and NG = 2: a block's vector instructions go from 542 to about
// 420, where they took 82% of the time; 16 x 8 key heads x 4 rows over 16384 keys
// then stream 4.3 TB/s, of the 4.95 that a large copy reaches.
template <bool F16, int D, int NG, bool EXACT, bool TREE = false>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attn_kv4_token_kernel(const KvAttnArgs p) {
    constexpr int GR = D / 64, DT = D / 16, NW = 4, RT = 16 / NG;
    __shared__ float xm[NW * NG][RT], xl[NW * NG][RT], xf[NW * NG][RT], xs[RT], xtop[RT];
    __shared__ __attribute__((aligned(16))) float xo[NW][16][D + 4];
    __shared__ u32x4 ql[NG * GR * 2][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, g = lane >> 4, own = col / RT;   // own: the block of the NG that the lane's column takes
    const int split = blockIdx.x % p.splits, bh = blockIdx.x / p.splits;
    const int b = bh / p.H, h = bh % p.H;
    const int R = p.G * p.Sq, row = min(col % RT, R - 1), qh = h * p.G + row / p.Sq, qt = row % p.Sq;

    const int len = p.valid ? min(max(p.valid[b], 0), p.Sk) : p.Sk;
    const int nblk = (len + kKvBlock - 1) / kKvBlock;   // the last token's row sees them all
    const int b0 = (int)((int64_t)nblk * split / p.splits), b1 = (int)((int64_t)nblk * (split + 1) / p.splits);
    const int lim_lo = TREE ? len - p.T : p.causal ? len - p.Sq + 1 : len;
    const int limit = !TREE && p.causal ? len - p.Sq + 1 + qt : len;

    const uint8_t* base = p.cache + (int64_t)bh * p.cache_blocks * Kv4<D>::kBytes;
    u32x4 kc[NG][GR], vc[NG][GR], kp[GR][2], vp[GR][2];
    auto load_keys = [&](int blk) __attribute__((always_inline)) {   // of blocks blk .. blk + NG - 1, the last one repeated
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int i = 0; i < GR; ++i)
                kc[n][i] = *reinterpret_cast<const u32x4*>(base + (int64_t)min(blk + n, b1 - 1) * Kv4<D>::kBytes + i * 1024 + lane * 16);
    };
    auto load_values = [&](int blk) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int i = 0; i < GR; ++i)
                vc[n][i] = *reinterpret_cast<const u32x4*>(base + (int64_t)min(blk + n, b1 - 1) * Kv4<D>::kBytes + Kv4<D>::kV + i * 1024 + lane * 16);
    };
    auto load_pars = [&](u32x4 (&par)[GR][2], int blk, int at) __attribute__((always_inline)) {   // of the own block
        const uint8_t* mine = base + (int64_t)min(blk + own, b1 - 1) * Kv4<D>::kBytes + at + 16 * g;
#pragma unroll
        for (int i = 0; i < GR; ++i)
#pragma unroll
            for (int t = 0; t < 2; ++t) par[i][t] = *reinterpret_cast<const u32x4*>(mine + (i * kKvBlock + 16 * t) * 4);
    };
    const int first = b0 + NG * wave;
    if (first < b1) {
        load_keys(first);
        load_pars(kp, first, Kv4<D>::kPar);
        load_pars(vp, first, Kv4<D>::kVPar);
        load_values(first);
    }

    u32x4 qf[GR][2];
    float qs[GR];
    kv_queries<F16, D>(p, b, qh, qt, g, qf, qs);
    float off[GR];
#pragma unroll
    for (int i = 0; i < GR; ++i) off[i] = EXACT ? -23.5f * qs[i] : 0.f, qs[i] *= p.scale_log2;
    if (wave < NG) {   // the queries of column group `wave`, zeros in the other columns
#pragma unroll
        for (int i = 0; i < GR; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) ql[(wave * GR + i) * 2 + k][lane] = own == wave ? qf[i][k] : u32x4{0, 0, 0, 0};
    }
    __syncthreads();

    f32x4 o[DT];   // O^T without the parameters' part pm
    float m = kKvNoMax, l = 0.f, pm[GR];
#pragma unroll
    for (int i = 0; i < GR; ++i) pm[i] = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const NibbleMask kmask = nibble_mask<F16>(), vmask = nibble_mask<false>();

    auto blocks = [&](const int blk, auto masked_c) __attribute__((always_inline)) {
        constexpr bool masked = decltype(masked_c)::value;
        const bool next = blk + NG * NW < b1;
        f32x4 s[2][GR];
#pragma unroll
        for (int i = 0; i < GR; ++i) s[0][i] = s[1][i] = f32x4{off[i], off[i], off[i], off[i]};
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int i = 0; i < GR; ++i)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32x4 q = ql[(n * GR + i) * 2 + k][lane];
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        s[t][i] = mfma_16b<F16>(nibbles_plus16<F16>(D == 64 ? kc[n][0][2 * t + k] : kc[n][t][2 * i + k], kmask), q, s[t][i]);
                }
        if (next) load_keys(blk + NG * NW);
        // scores less the row's maximum, base 2
        const int key0 = kKvBlock * (blk + own) + 4 * g;
        uint32_t see = 0xffu;
        if (masked) {
            see = 0;
            if (blk + own < b1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int key = key0 + 16 * (e >> 2) + (e & 3);
                    if (key < limit && (!p.mask || p.mask[b * p.mask_stride + key])) see |= 1u << e;
                }
                if (TREE) see &= kv_lane_bits(kv_tree_bits(p, b, p.T - p.Sq + qt, kKvBlock * (blk + own), len - p.T), g);
            }
        }
        float x[8];
        const float neg = m == kKvNoMax ? 0.f : -m;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float u = neg;
#pragma unroll
            for (int i = 0; i < GR; ++i) {
                uint32_t k = kp[i][e >> 2][e & 3];
                if (masked && !(see >> e & 1u)) k = 0u;   // what the row does not see may hold anything
                u = __builtin_fmaf(__uint_as_float(k << 16) * p.scale_log2, s[e >> 2][i][e & 3], __builtin_fmaf(EXACT ? __uint_as_float(k & 0xffff0000u) : kv_mix(k, -23.5f, 1.f), qs[i], u));
            }
            x[e] = masked && !(see >> e & 1u) ? -INFINITY : u;
        }
        if (next) load_pars(kp, blk + NG * NW, Kv4<D>::kPar);
        const float mx = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__any(mx > (m == kKvNoMax ? -INFINITY : kKvSlack))) {
            const float al = kv_raise(x, mx, m);
            l *= al;
#pragma unroll
            for (int i = 0; i < GR; ++i) pm[i] *= al;
#pragma unroll
            for (int i = 0; i < DT; ++i) o[i] *= al;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[e] = __builtin_amdgcn_exp2f(x[e]);
            l += x[e];
        }
#pragma unroll
        for (int i = 0; i < GR; ++i) {
            u32x4 hi, lo, rest;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t v0 = vp[i][e >> 1][2 * (e & 1)], v1 = vp[i][e >> 1][2 * (e & 1) + 1];
                if (masked && !(see >> (2 * e) & 1u)) v0 = 0u;
                if (masked && !(see >> (2 * e + 1) & 1u)) v1 = 0u;
                float a = x[2 * e] * __uint_as_float(v0 << 16), c = x[2 * e + 1] * __uint_as_float(v1 << 16);
                const uint32_t w = pack_bf16x2(a, c);
                a -= __uint_as_float(w << 16), c -= __uint_as_float(w & 0xffff0000u);
                const uint32_t r = pack_bf16x2(a, c);
                pm[i] += x[2 * e] * __uint_as_float(v0 & 0xffff0000u) + x[2 * e + 1] * __uint_as_float(v1 & 0xffff0000u);
                if (!EXACT) pm[i] = kv_dot(w, kv_dot(r, pm[i]));
                hi[e] = w;
                lo[e] = r;
                if (EXACT) rest[e] = pack_bf16x2(a - __uint_as_float(r << 16), c - __uint_as_float(r & 0xffff0000u));
            }
#pragma unroll
            for (int d = 4 * i; d < 4 * i + 4; ++d)
                if (EXACT) o[d] = mfma_16b<false>(kv_offset(), hi, o[d]);
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const uint32_t keep = own == n ? 0xffffffffu : 0u;
                const u32x4 ph = hi & keep, pl = lo & keep;   // the weights of block n, zeros in the other columns
#pragma unroll
                for (int t = 2 * i; t < 2 * i + 2; ++t) {
                    const uint32_t w0 = vc[n][t >> 1][2 * (t & 1)], w1 = vc[n][t >> 1][2 * (t & 1) + 1];
                    const u32x4 va = {nibble_pair_plus16<false, 0>(w0, vmask), nibble_pair_plus16<false, 2>(w0, vmask),
                                      nibble_pair_plus16<false, 0>(w1, vmask), nibble_pair_plus16<false, 2>(w1, vmask)};
                    const u32x4 vb = {nibble_pair_plus16<false, 1>(w0, vmask), nibble_pair_plus16<false, 3>(w0, vmask),
                                      nibble_pair_plus16<false, 1>(w1, vmask), nibble_pair_plus16<false, 3>(w1, vmask)};
                    o[2 * t] = mfma_16b<false>(va, pl, mfma_16b<false>(va, ph, o[2 * t]));
                    o[2 * t + 1] = mfma_16b<false>(vb, pl, mfma_16b<false>(vb, ph, o[2 * t + 1]));
                    if (EXACT) {
                        o[2 * t] = mfma_16b<false>(va, rest & keep, o[2 * t]);
                        o[2 * t + 1] = mfma_16b<false>(vb, rest & keep, o[2 * t + 1]);
                    }
                }
            }
#pragma unroll
            for (int d = 4 * i; d < 4 * i + 4; ++d)   // the small terms where the sum is small again
                if (EXACT) o[d] = mfma_16b<false>(kv_offset(), rest, mfma_16b<false>(kv_offset(), lo, o[d]));
        }
        if (next) {
            load_pars(vp, blk + NG * NW, Kv4<D>::kVPar);
            load_values(blk + NG * NW);
        }
    };
    for (int blk = first; blk < b1; blk += NG * NW) {
        if (p.mask || blk + NG > b1 || kKvBlock * (blk + NG) > lim_lo) blocks(blk, std::true_type{});
        else blocks(blk, std::false_type{});
    }

    // Waves and column groups meet.
    l = lanes4_sum(l);
#pragma unroll
    for (int i = 0; i < GR; ++i) {
        const float add = lanes4_sum(pm[i]);
#pragma unroll
        for (int d = 4 * i; d < 4 * i + 4; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[d][e] += add;
    }
    if (g == 0) xm[wave * NG + own][col % RT] = m, xl[wave * NG + own][col % RT] = l;
    __syncthreads();
    if (threadIdx.x < RT) {
        const int i = threadIdx.x;
        float top = xm[0][i], sum = 0.f;
#pragma unroll
        for (int w = 1; w < NW * NG; ++w) top = fmaxf(top, xm[w][i]);
#pragma unroll
        for (int w = 0; w < NW * NG; ++w) {
            const float f = __builtin_amdgcn_exp2f(xm[w][i] - top);
            xf[w][i] = f;
            sum += f * xl[w][i];
        }
        xs[i] = sum;
        xtop[i] = top;
    }
    __syncthreads();
    const float f = xf[wave * NG + own][col % RT];
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&xo[wave][col][16 * d + 4 * g]) = o[d] * f;
    __syncthreads();
    constexpr int E = RT * D / 256 > 2 ? RT * D / 256 : 2;   // channels a thread finishes
    const int r = (int)threadIdx.x / (D / E), d0 = E * ((int)threadIdx.x % (D / E));
    if (r >= RT || r >= R) return;
    float y[E];
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] += xo[w][n * RT + r][d0 + e];
    kv_finish<D, E>(p, split, b, h * p.G + r / p.Sq, r % p.Sq, d0, y, xtop[r], xs[r]);
}

// out = sum_splits O 2^(m - M) / sum_splits l 2^(m - M), a workgroup for each row
// whose four waves deal the splits: all of a row's loads are in flight at once
// (with one wave to a row, eight splits at a time, 32 rows of 20 splits took 3.6
// us).
template <int D>
__global__ __launch_bounds__(256) void attn_kv4_merge_kernel(const KvAttnArgs p) {
    constexpr int E = D / 64, kEach = kKvMaxSplits / 4;
    __shared__ float part[4][D];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t row = blockIdx.x;
    const float* src = p.part + row * (D + 2);
    const int64_t step = p.rows * (D + 2);
    float m = kKvNoMax, l = 0.f, v[kEach][E];
    if (lane < p.splits) m = src[lane * step + D], l = src[lane * step + D + 1];
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        if (wave + 4 * j < p.splits)
#pragma unroll
            for (int e = 0; e < E; ++e) v[j][e] = src[(wave + 4 * j) * step + 64 * e + lane];
    float mm = m;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o, 64));
    const float w = __builtin_amdgcn_exp2f(m - mm);   // l is 0 behind the last split
    float sum = l * w;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        if (wave + 4 * j < p.splits) {
            const float ws = __shfl(w, wave + 4 * j, 64);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += ws * v[j][e];
        }
#pragma unroll
    for (int e = 0; e < E; ++e) part[wave][64 * e + lane] = acc[e];
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= D) return;
    const float y = (part[0][d] + part[1][d] + part[2][d] + part[3][d]) * (sum == 0.f ? 0.f : 1.f / sum);
    const int s = (int)(row % p.Sq);
    const int64_t bh = row / p.Sq, Hq = (int64_t)p.H * p.G;
    const int64_t i = bh / Hq * p.os[0] + bh % Hq * p.os[1] + s * p.os[2] + d;
    if (p.out_kind == 0) static_cast<float*>(p.out)[i] = y;
    else if (p.out_kind == 1) static_cast<uint16_t*>(p.out)[i] = (uint16_t)f32_to_bf16_bits(y);
    else static_cast<_Float16*>(p.out)[i] = (_Float16)y;
}

// How a call is cut up: tiles of 16 query rows to a workgroup (qt), groups of
// them (qgroups), key splits; and how p and V meet.
struct KvPlan {
    int qt, ng, qgroups, splits, form;
    int64_t wgs, rows;
};

static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

static inline int kv_form(const sf_attn_kv4_desc* d, bool tree) {   // with more than one tile of rows
    const bool apart = tree || (d->is_causal && d->Sq > 1);   // rows that see different tokens
    return d->out_dtype == SF_F32 ? kKvExact : d->out_dtype == SF_F16 || apart || d->exact_pv ? kKvPair : kKvHalf;
}

// Up to 16 rows to a key head: one tile, four waves to a workgroup.  Up to 512
// keys a wave has four blocks at most and a merge costs what it saves (us with
// one split and four, 512 keys: 8 heads of 128 channels 8.0 and 7.4, 16 x 8 heads
// 8.6 and 9.6, 8 x 8 of 64 5.8 and 6.7; 700 keys, 8 heads: 10.6 and 8.9); beyond,
// about two workgroups a CU of at least a block to a wave, and no split over 2048
// keys, so that batches of unequal lengths spread (16 x 8 heads, 4096..16384
// keys: 59 us with 8 splits, 58 with 4, 148 with 1).
static int kv_splits_one_tile(const sf_attn_kv4_desc* d, int64_t base) {
    if (d->Sk <= 512 || (int64_t)d->B * d->Hq * d->Sq >= kKvMergeRows) return 1;
    const int64_t want = std::max(ceil_div(512, base), ceil_div(d->Sk, 2048));
    return (int)std::min<int64_t>({want, ceil_div(d->Sk, 128), (int64_t)kKvMaxSplits});
}

// Column groups of one tile (attn_kv4_token_kernel; 1: attn_kv4_kernel): where
// there are enough blocks of keys, 16 for each SIMD, that the vector units and
// the stream bound the call and not its start.  us, with 1, 2 and 4 groups: 8 x
// 32 heads x 8192 keys of 64 channels 45, 41, 37; 16 x 8 x 16384 of 128, four rows
// each, 77 and 70 (four groups would spill); 8 x 8 x 4096 17.2 and 16.9; 16 x 8 x
// 1024 13.0 and 13.4.
static int kv_column_groups(const sf_attn_kv4_desc* d, int rows, int64_t heads) {
    if (rows > 8 || heads * ceil_div(d->Sk, kKvBlock) < 16384) return 1;
    return d->cache.D == 64 && rows <= 4 ? 4 : 2;
}

// More rows: a workgroup holds a CU alone, so the time is its rounds times what
// one takes: per wave and block of 32 keys `step` us times (1.5 + qt) -- the
// block's unpacking, then each tile -- and 3 + 0.8 qt us around the loop; key
// splits that fill the card add a merge of 7 us.  Estimated for each qt the
// kernel is built for, the smallest taken.  Measured against it (64 channels,
// bf16): 32 x 67 rows x 4374 keys 20.1 us with qt 3 and four splits, 21.1 with 5 and
// eight, 32 with 3 and one (estimates 19, 20, 30); 256 x 67 x 4374 42 with qt 5, 64
// with 3; 256 x 67 x 67 9.8 with qt 5, 13.8 with 3.  The (hi, lo) form takes 0.42 us
// a step, and qt 5 would spill, with three terms qt 4: causal, 12 x 520 rows x 1537
// keys 16.2 with qt 2, 19.4 with 3, 23 with 4; 16 x 1024 x 2048 26.7 with 4, 35 with
// 2.  128 channels: 2 tiles are what fits; a step of theirs takes about half as long again as `step` (16 x 8 heads of 64
// rows over up to 8192 keys: 52 by this, 79 measured), which only the splits of few workgroups go by.
static void kv_tiles(const sf_attn_kv4_desc* d, int64_t R, int64_t heads, KvPlan& k) {
    const bool wide = d->cache.D == 128;
    const int most = wide ? 2 : k.form == kKvExact ? 3 : k.form == kKvPair ? 4 : 5;
    const int64_t per_block = kKvBlock * 8;   // a block to each wave
    const double step = k.form == kKvHalf ? 0.3 : 0.42;
    double best = 0.;
    for (int qt = 2; qt <= most; ++qt) {
        const int64_t groups = ceil_div(R, 16 * qt), base = heads * groups;
        const int64_t fill = std::min<int64_t>(base < 256 ? 256 / base : 1, kKvMaxSplits);
        for (int64_t s = 1; s <= fill; s += fill > 1 ? fill - 1 : 1) {
            const int64_t splits = d->num_splits > 0 ? d->num_splits : std::min(s, std::max<int64_t>(1, ceil_div(d->Sk, per_block)));
            const double us = (double)ceil_div(base * splits, 256) *
                                  ((double)ceil_div(d->Sk, per_block * splits) * step * (1.5 + qt) + 3. + 0.8 * qt) +
                              (splits > 1 ? 7. : 0.);
            if (best == 0. || us < best) {
                best = us;
                k.qt = qt;
                k.qgroups = (int)groups;
                k.splits = (int)splits;
            }
        }
    }
}

static KvPlan kv_plan(const sf_attn_kv4_desc* d, bool tree) {
    KvPlan k = {};
    const int64_t R = (int64_t)(d->Hq / d->cache.H) * d->Sq, heads = (int64_t)d->B * d->cache.H;
    k.rows = (int64_t)d->B * d->Hq * d->Sq;
    k.form = kv_form(d, tree);
    if (R <= 16) {
        k.qt = k.qgroups = 1;
        k.splits = d->num_splits > 0 ? d->num_splits : kv_splits_one_tile(d, heads);
        k.ng = kv_column_groups(d, (int)R, heads);
    } else {
        kv_tiles(d, R, heads, k);
        if (k.form == kKvHalf && ceil_div(d->Sk, 8 * k.splits) > kKvHalfKeys) {
            k.form = kKvPair;
            kv_tiles(d, R, heads, k);
        }
    }
    k.wgs = heads * k.qgroups * k.splits;
    return k;
}

static int kv_attn_check(const sf_attn_kv4_desc* d) {
    if (!d || d->B < 0 || d->Hq < 0 || d->Sq < 0 || d->Sk < 0 || d->cache.B <= 0 || d->cache.H <= 0 ||
        d->cache.capacity <= 0)
        return SF_EINVAL;
    if (d->cache.D != 64 && d->cache.D != 128) return SF_ENOTSUP;
    if (d->Hq % d->cache.H || d->B != d->cache.B || d->Sk > d->cache.capacity) return SF_EINVAL;
    if (d->num_splits < 0 || d->num_splits > kKvMaxSplits) return SF_EINVAL;
    if (d->Sk > 1 << 30 || (int64_t)d->Hq / d->cache.H * d->Sq > 1 << 30) return SF_ENOTSUP;   // counted in 32 bits
    return SF_OK;
}

static size_t kv_workspace(const sf_attn_kv4_desc* d, bool tree) {
    const KvPlan k = kv_plan(d, tree);
    return k.splits > 1 ? (size_t)k.splits * (size_t)k.rows * (d->cache.D + 2) * sizeof(float) : 0;
}

static int kv_tree_check(const sf_attn_kv4_desc* d, const sf_draft_tree* tree) {
    if (!tree || d->is_causal || tree->T <= 0 || d->Sq > tree->T) return SF_EINVAL;
    if (tree->T > SF_TREE_MAX_NODES) return SF_ENOTSUP;
    return SF_OK;
}

template <bool F16, bool TREE>
static void kv_launch(const KvAttnArgs& p, const KvPlan& k, int D, hipStream_t s) {
    const dim3 grid((unsigned)k.wgs);
#define SF_KV4_LAUNCH(DD, QT, FORM, NW) \
    hipLaunchKernelGGL((attn_kv4_kernel<F16, DD, QT, FORM, NW, TREE>), grid, dim3(64 * NW), 0, s, p)
#define SF_KV4_TOKEN(DD, NG, EXACT) hipLaunchKernelGGL((attn_kv4_token_kernel<F16, DD, NG, EXACT, TREE>), grid, dim3(256), 0, s, p)
    const int form = k.form;
    if (k.qt == 1 && form == kKvExact) {
        if (D == 64) {
            if (k.ng == 1) SF_KV4_LAUNCH(64, 1, kKvExact, 4);
            else if (k.ng == 2) SF_KV4_TOKEN(64, 2, true);
            else SF_KV4_TOKEN(64, 4, true);
        } else {
            if (k.ng == 1) SF_KV4_LAUNCH(128, 1, kKvExact, 4);
            else SF_KV4_TOKEN(128, 2, true);
        }
    } else if (k.qt == 1) {
        if (D == 64) {
            if (k.ng == 1) SF_KV4_LAUNCH(64, 1, kKvPair, 4);
            else if (k.ng == 2) SF_KV4_TOKEN(64, 2, false);
            else SF_KV4_TOKEN(64, 4, false);
        } else {
            if (k.ng == 1) SF_KV4_LAUNCH(128, 1, kKvPair, 4);
            else SF_KV4_TOKEN(128, 2, false);
        }
    } else if (form == kKvExact) {
        if (D == 128) SF_KV4_LAUNCH(128, 2, kKvExact, 8);
        else if (k.qt == 2) SF_KV4_LAUNCH(64, 2, kKvExact, 8);
        else SF_KV4_LAUNCH(64, 3, kKvExact, 8);
    } else if (form == kKvPair) {
        if (D == 128) SF_KV4_LAUNCH(128, 2, kKvPair, 8);
        else if (k.qt == 2) SF_KV4_LAUNCH(64, 2, kKvPair, 8);
        else if (k.qt == 3) SF_KV4_LAUNCH(64, 3, kKvPair, 8);
        else SF_KV4_LAUNCH(64, 4, kKvPair, 8);
    } else if constexpr (!TREE) {
        if (D == 128) SF_KV4_LAUNCH(128, 2, kKvHalf, 8);
        else if (k.qt == 2) SF_KV4_LAUNCH(64, 2, kKvHalf, 8);
        else if (k.qt == 3) SF_KV4_LAUNCH(64, 3, kKvHalf, 8);
        else if (k.qt == 4) SF_KV4_LAUNCH(64, 4, kKvHalf, 8);
        else SF_KV4_LAUNCH(64, 5, kKvHalf, 8);
    }
#undef SF_KV4_TOKEN
#undef SF_KV4_LAUNCH
}

static int kv_attn(const sf_attn_kv4_desc* d, const sf_draft_tree* tree, const void* q, void* out, void* workspace,
                   size_t workspace_bytes, void* stream) {
    if (!d->B || !d->Hq || !d->Sq) return SF_OK;
    if (d->in_dtype != SF_BF16 && d->in_dtype != SF_F16) return SF_ENOTSUP;
    if (d->out_dtype != SF_BF16 && d->out_dtype != SF_F16 && d->out_dtype != SF_F32) return SF_ENOTSUP;
    if (d->scale < 0.f) return SF_ENOTSUP;
    if (!q || !out || !d->cache.data) return SF_EINVAL;
    if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(d->cache.data)) & 15)
        return SF_EINVAL;
    for (int i = 0; i < 3; ++i)
        if (d->q_stride[i] < 0 || (d->q_stride[i] & 7) || d->o_stride[i] < 0 || (d->o_stride[i] & 7)) return SF_EINVAL;
    if (d->kv_mask && d->kv_mask_stride < 0) return SF_EINVAL;
    const KvPlan k = kv_plan(d, tree != nullptr);
    if (k.wgs >= 1 << 23 || (k.splits > 1 && k.rows >= kKvMergeRows)) return SF_ENOTSUP;   // threads in 32 bits
    if (k.splits > 1 && (!workspace || workspace_bytes < kv_workspace(d, tree != nullptr))) return SF_EWORKSPACE;
    if (k.splits > 1 && (reinterpret_cast<uintptr_t>(workspace) & 3)) return SF_EINVAL;
    KvAttnArgs p = {};
    p.q = static_cast<const uint16_t*>(q);
    p.cache = static_cast<const uint8_t*>(d->cache.data);
    p.out = out;
    p.part = static_cast<float*>(workspace);
    p.valid = d->kv_valid_len;
    p.mask = d->kv_mask;
    p.mask_stride = d->kv_mask_stride;
    p.cache_blocks = kv4_blocks(d->cache.capacity);
    for (int i = 0; i < 3; ++i) p.qs[i] = d->q_stride[i], p.os[i] = d->o_stride[i];
    p.rows = k.rows;
    p.B = d->B;
    p.H = d->cache.H;
    p.G = d->Hq / d->cache.H;
    p.Sq = d->Sq;
    p.Sk = d->Sk;
    p.splits = k.splits;
    p.qgroups = k.qgroups;
    p.causal = d->is_causal != 0;
    p.out_kind = d->out_dtype == SF_BF16 ? 1 : (d->out_dtype == SF_F16 ? 2 : 0);
    p.scale_log2 = (d->scale == 0.f ? 1.f / sqrtf((float)d->cache.D) : d->scale) * 1.4426950408889634f;
    if (tree) {
        p.tree = tree->masks;
        p.T = tree->T;
        p.tree_words = (tree->T + 31) / 32;
        p.tree_stride = tree->each ? (int64_t)p.T * p.tree_words : 0;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const bool f16 = d->in_dtype == SF_F16;
    if (tree) {
        if (f16) kv_launch<true, true>(p, k, d->cache.D, s);
        else kv_launch<false, true>(p, k, d->cache.D, s);
    } else {
        if (f16) kv_launch<true, false>(p, k, d->cache.D, s);
        else kv_launch<false, false>(p, k, d->cache.D, s);
    }
    if (hipGetLastError() != hipSuccess) return SF_ELAUNCH;
    if (k.splits > 1) {
        const dim3 mg((unsigned)k.rows);
        if (d->cache.D == 64) hipLaunchKernelGGL(attn_kv4_merge_kernel<64>, mg, dim3(256), 0, s, p);
        else hipLaunchKernelGGL(attn_kv4_merge_kernel<128>, mg, dim3(256), 0, s, p);
        if (hipGetLastError() != hipSuccess) return SF_ELAUNCH;
    }
    return SF_OK;
}

}  // namespace sfk

extern "C" size_t sf_attn_kv4_workspace_bytes(const sf_attn_kv4_desc* d) {
    if (sfk::kv_attn_check(d) != SF_OK || !d->B || !d->Hq || !d->Sq) return 0;
    return sfk::kv_workspace(d, false);
}

extern "C" int sf_attn_kv4(const sf_attn_kv4_desc* d, const void* q, void* out, void* workspace, size_t workspace_bytes,
                           void* stream) {
    const int st = sfk::kv_attn_check(d);
    return st != SF_OK ? st : sfk::kv_attn(d, nullptr, q, out, workspace, workspace_bytes, stream);
}

extern "C" size_t sf_attn_kv4_tree_workspace_bytes(const sf_attn_kv4_desc* d, const sf_draft_tree* tree) {
    if (sfk::kv_attn_check(d) != SF_OK || sfk::kv_tree_check(d, tree) != SF_OK || !d->B || !d->Hq || !d->Sq) return 0;
    return sfk::kv_workspace(d, true);
}

extern "C" int sf_attn_kv4_tree(const sf_attn_kv4_desc* d, const sf_draft_tree* tree, const void* q, void* out,
                                void* workspace, size_t workspace_bytes, void* stream) {
    int st = sfk::kv_attn_check(d);
    if (st == SF_OK) st = sfk::kv_tree_check(d, tree);
    if (st != SF_OK) return st;
    if (!tree->masks || (reinterpret_cast<uintptr_t>(tree->masks) & 3)) return SF_EINVAL;
    return sfk::kv_attn(d, tree, q, out, workspace, workspace_bytes, stream);
}
