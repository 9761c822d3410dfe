// Projections over 4-bit weights with group scales (gfx950).
//
// C[m][n] = act(sum_k A[m][k] s[n][k / g] (c[n][k] - z[n][k / g]) + bias[n]),
// codes c in 0..15.  A code goes into a 16-bit matrix operand without an
// arithmetic conversion: its four bits are placed at the top of the mantissa
// of 16.0, which makes the operand 16 + c exactly (bf16 0x4180 | c << 3, fp16
// 0x4C00 | c << 6), two codes for one shift and one and-or.  The products with
// A are exact in the fp32 accumulator, and a group ends with
//   acc += s (sum_k (16 + c) A - (16 + z) sum_k A),
// sum_k A of the group from one more matrix product with an operand of ones.
// Scale and zero point never round to 16 bits; the offset of 16 costs the
// accumulator about two bits (the sums are of 16..31 instead of -8..7).
//
// Layout (sf_w4_pack): blocks of 16 rows x 128 columns, 1 KB each, lane
// l = 16 g + r of a wave holding row r's codes k = 32 j + 8 g + e in dword j,
// code e at nibble (e >> 1) + 4 (e & 1): one 16-byte load per lane is the
// operand of four v_mfma_f32_16x16x32.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sf_act.h"
#include "sf_device.h"
#include "sf_hip.h"
#include "sf_nibble.h"

namespace sfk {

struct W4Args {
    const uint16_t* a;     // [M][lda]
    int64_t lda;
    const uint8_t* w;      // packed codes, then params
    const uint32_t* par;   // [N16][groups][16]: scale bits << 16 | zero
    const float* bias;
    void* c;
    int64_t ldc;
    int M, N, K, KB, groups, n16;
    int scale_f16, act, c_kind, accumulate;
    int vec4;              // four columns of C fit one aligned store
};

__device__ __forceinline__ float w4_scale(uint32_t u, int f16) {
    return f16 ? (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16)) : __uint_as_float(u & 0xffff0000u);
}

// A wave's operands of one block of 128 inputs: codes and parameters of its NT
// tiles of 16 rows of W.
template <int NT, int GROUPS>
struct W4Block {
    u32x4 code[NT], par[NT][GROUPS];
};

// Four columns of a row of C, from column n.
__device__ __forceinline__ void w4_store(const W4Args& p, int m, int n, f32x4 v) {
    if (m >= p.M || n >= p.N) return;
    const int64_t at = (int64_t)m * p.ldc + n;
    const int cols = min(4, p.N - n);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < cols) v[i] = apply_act(p.act, v[i] + (p.bias ? p.bias[n + i] : 0.f));
    if (cols == 4 && p.vec4) {
        if (p.c_kind == 0) {
            f32x4* c = reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + at);
            *c = p.accumulate ? *c + v : v;
        } else {
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.c) + at) =
                p.c_kind == 1 ? uint2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])}
                              : uint2{pack_f16x2_rn(v[0], v[1]), pack_f16x2_rn(v[2], v[3])};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= cols) continue;
        if (p.c_kind == 0) {
            float* c = static_cast<float*>(p.c) + at + i;
            *c = p.accumulate ? *c + v[i] : v[i];
        } else if (p.c_kind == 1) {
            static_cast<uint16_t*>(p.c)[at + i] = (uint16_t)f32_to_bf16_bits(v[i]);
        } else {
            static_cast<_Float16*>(p.c)[at + i] = (_Float16)v[i];
        }
    }
}

// One workgroup: 16 MB rows x 16 NT WN columns.  Its eight waves take NT tiles of
// columns each and deal the blocks of 128 inputs among 8 / WN; the sums meet in
// LDS.  A wave brings its activations into LDS itself, straight from memory: with
// one or two waves to a SIMD that is what keeps a block in flight while another
// is computed (through registers 67 x 6144 x 2048 took 14 us, and 10.2 so), and
// pieces of 16 bytes are placed so that neither side meets in a bank.  WN = 2: the
// waves of two column tiles bring half of each block and read it both, for which
// they meet at a barrier; the blocks alternate between two places.
template <bool F16, int MB, int NT, int WN, int GROUP>
__global__ __launch_bounds__(512) void gemm_w4_kernel(const W4Args p) {
    constexpr int WK = 8 / WN, kSteps = GROUP / 32, kGroups = 4 / kSteps, kStage = 16 * MB * 256;
    __shared__ __attribute__((aligned(1024))) char lds[8 * kStage];
    static_assert(MB * NT * 1024 <= kStage, "the sums take the place of the activations");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int wk = wave / WN, wn = wave % WN;
    const int nb0 = (blockIdx.x * WN + wn) * NT, m0 = blockIdx.y * 16 * MB, rows = min(16 * MB, p.M - m0);
    const uint32_t ld = 2u * (uint32_t)p.lda;   // bytes: lda is at most 2^23
    const __amdgpu_buffer_rsrc_t ars = make_rsrc(p.a + (int64_t)m0 * p.lda, (uint32_t)rows * ld);
    char* stage = lds + wk * WN * kStage;   // WN of them, in turn
    // Instruction i brings rows 4 i .. 4 i + 3, 256 bytes each, piece c of row q to place c ^ (q & 15); rows behind M are
    // behind the buffer's end and come as zeros.
    auto fetch = [&](int kb, char* to) __attribute__((always_inline)) {
        // A last block that is not full: one of its groups again in the places of the missing ones, whose scale is 0 (0
        // times a finite sum, as the group's own is).
        const int have = GROUP < 128 ? min(16, (p.K - 128 * kb) >> 3) : 16;
        uint32_t at[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            int c = r ^ ((4 * (u + wn * (4 * MB / WN)) & 15) + g);
            if (GROUP == 64) c &= have - 1;                               // 8 or 16 of them
            if (GROUP == 32) c = c < have ? c : have == 12 ? c & 11 : c & (have - 1);
            at[u] = (uint32_t)g * ld + 16u * (uint32_t)c;
        }
        uint32_t step = 256u * (uint32_t)kb + (uint32_t)wn * (4 * MB / WN) * 4u * ld;
        to += wn * (4 * MB / WN) * 1024;
#pragma unroll
        for (int i = 0; i < 4 * MB / WN; ++i) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(ars, (__attribute__((address_space(3))) void*)(to + 1024 * i), 16,
                                                     at[i & 3] + step, 0, 0, 0);
            step += 4u * ld;
        }
    };
    const uint8_t* wtile[NT];
    const uint32_t* ptile[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {   // tiles behind the last one repeat it; they are not stored
        const int64_t nb = min(nb0 + t, p.n16 - 1);
        wtile[t] = p.w + nb * p.KB * 1024 + 16 * lane;
        ptile[t] = p.par + nb * p.groups * 16 + 4 * g;
    }
    auto load_w = [&](W4Block<NT, kGroups>& o, int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            o.code[t] = *reinterpret_cast<const u32x4*>(wtile[t] + (int64_t)kb * 1024);
#pragma unroll
            for (int q = 0; q < kGroups; ++q)
                o.par[t][q] = *reinterpret_cast<const u32x4*>(ptile[t] + (int64_t)(kb * kGroups + q) * 16);
        }
    };
    f32x4 acc[NT][MB];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = f32x4{0.f, 0.f, 0.f, 0.f};
    const NibbleMask nmask = nibble_mask<F16>();
    const u32x4 ones = F16 ? u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u}
                           : u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
    W4Block<NT, kGroups> cur, nxt;
    if (wk < p.KB) {
        load_w(nxt, wk);
        fetch(wk, stage);
    }
    int turn = 0;
    for (int kb = wk; (WN > 1 ? kb - wk : kb) < p.KB; kb += WK, turn = WN - 1 - turn) {
        cur = nxt;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (WN > 1) {
            __syncthreads();
            if (kb >= p.KB) break;   // the last round of some waves
        }
        const char* from = stage + turn * kStage;
        u32x4 x[MB][4];
#pragma unroll
        for (int b = 0; b < MB; ++b)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[b][j] = *reinterpret_cast<const u32x4*>(from + (16 * b + r) * 256 + 16 * ((4 * j + g) ^ r));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next block is brought into its place
        if (kb + WK < p.KB) {
            load_w(nxt, kb + WK);
            fetch(kb + WK, stage + (WN - 1 - turn) * kStage);
        }
#pragma unroll
        for (int q = 0; q < kGroups; ++q) {
            f32x4 sx[MB];
#pragma unroll
            for (int b = 0; b < MB; ++b) sx[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = q * kSteps; j < (q + 1) * kSteps; ++j)
#pragma unroll
                for (int b = 0; b < MB; ++b) sx[b] = mfma_16b<F16>(ones, x[b][j], sx[b]);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                f32x4 pr[MB];
#pragma unroll
                for (int b = 0; b < MB; ++b) pr[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = q * kSteps; j < (q + 1) * kSteps; ++j) {
                    const u32x4 w = nibbles_plus16<F16>(cur.code[t][j], nmask);
#pragma unroll
                    for (int b = 0; b < MB; ++b) pr[b] = mfma_16b<F16>(w, x[b][j], pr[b]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t par = cur.par[t][q][i];
                    const float sc = w4_scale(par, p.scale_f16), z = 16.f + (float)(par & 0xffu);
#pragma unroll
                    for (int b = 0; b < MB; ++b)
                        acc[t][b][i] = __builtin_fmaf(sc, __builtin_fmaf(-z, sx[b][0], pr[b][i]), acc[t][b][i]);
                }
            }
        }
    }
    __syncthreads();
    f32x4* red = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) red[(wave * NT * MB + t * MB + b) * 64 + lane] = acc[t][b];
    __syncthreads();
    for (int u = wk; u < NT * MB; u += WK) {
        f32x4 v = red[(wn * NT * MB + u) * 64 + lane];
#pragma unroll
        for (int w = 1; w < WK; ++w) v += red[((w * WN + wn) * NT * MB + u) * 64 + lane];
        w4_store(p, m0 + 16 * (u % MB) + r, 16 * (nb0 + u / MB) + 4 * g, v);
    }
}

// One thread per dword of the packed codes, then one per parameter.
__global__ __launch_bounds__(256) void w4_pack_kernel(const sf_w4_pack_desc d, uint32_t* out, int n16, int KB,
                                                      int groups) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t codes = (int64_t)n16 * KB * 256;
    if (i < codes) {
        const int j = i & 3, l = (i >> 2) & 63;
        const int64_t blk = i >> 8;
        const int64_t n = blk / KB * 16 + (l & 15);
        const int k = (int)(blk % KB) * 128 + 32 * j + 8 * (l >> 4);
        uint32_t v = 0;
        if (n < d.N && k < d.K) {
#pragma unroll
            for (int b = 0; b < 4; ++b) {   // byte b: codes 2 b and 2 b + 1, at nibbles b and b + 4
                const uint32_t two = d.codes[n * d.ldc + (k >> 1) + b];
                v |= (two & 15u) << (4 * b) | (two >> 4) << (16 + 4 * b);
            }
        }
        out[i] = v;
    } else if (i < codes + (int64_t)n16 * groups * 16) {
        const int64_t q = i - codes;
        const int64_t n = q / ((int64_t)groups * 16) * 16 + (q & 15);
        const int gr = (int)((q >> 4) % groups);
        uint32_t v = 0;
        if (n < d.N && gr < d.K / d.group) {
            const uint32_t s = static_cast<const uint16_t*>(d.scales)[n * d.lds + gr];
            v = s << 16 | (d.zeros ? d.zeros[n * d.ldz + gr] : 8u);
        }
        out[i] = v;
    }
}

static inline bool w4_shape_ok(int32_t N, int32_t K, int32_t group) {
    return N > 0 && K > 0 && (group == 32 || group == 64 || group == 128) && K % group == 0;
}
static inline int w4_kb(int K) { return (K + 127) / 128; }
static inline int w4_groups(int K, int group) { return w4_kb(K) * (128 / group); }

template <bool F16, int MB, int NT, int WN, int GROUP>
static void launch_w4_shape(const W4Args& p, hipStream_t s) {
    const dim3 grid((unsigned)((p.n16 + NT * WN - 1) / (NT * WN)), (unsigned)((p.M + 16 * MB - 1) / (16 * MB)));
    hipLaunchKernelGGL((gemm_w4_kernel<F16, MB, NT, WN, GROUP>), grid, dim3(512), 0, s, p);
}

// The shape whose estimate is the smallest: rounds of 256 workgroups, each 0.5 us
// and for every block of 128 inputs of a wave 0.2 + 0.25 MB NT - 0.1 MB (WN - 1).
// Fitted to 63 products of 8..536 rows, 2048..16384 columns and 2048..8192 inputs
// with the weights from memory, where the choice costs 3% in the mean, and up to a
// third, over the fastest of 16 shapes.  us, MB,NT,WN:
//   16 x 2048 x 2048: 3.9 with 1,1,1, 4.9 with 1,2,1; 16 x 8192 x 8192: 11.0 with 1,2,1, 14.6 with 1,1,1;
//   32 x 8192 x 8192: 14.8 with 2,2,1, 17.7 with 1,2,1; 48 x 6144 x 2048: 8.0 with 3,2,1, 10.1 with 2,2,1;
//   67 x 6144 x 2048: 10.6 with 5,2,1, 13.1 with 3,2,1; 536 x 8192 x 2048: 46.7 with 5,2,2, 57.2 with 5,2,1.
// Groups of 32 keep four times the parameters; five tiles of rows do not fit the registers beside them.
template <bool F16, int GROUP>
static void launch_w4(const W4Args& p, hipStream_t s) {
    static const int shapes[6][3] = {{1, 1, 1}, {1, 2, 1}, {2, 2, 1}, {3, 2, 1}, {5, 2, 1}, {5, 2, 2}};
    int best = 0;
    double least = 0.;
    for (int i = 0; i < (GROUP == 32 ? 4 : 6); ++i) {
        const int mb = shapes[i][0], nt = shapes[i][1], wn = shapes[i][2];
        const int64_t slabs = ((int64_t)p.M + 16 * mb - 1) / (16 * mb), wgs = slabs * ((p.n16 + nt * wn - 1) / (nt * wn));
        if (slabs > 65535) continue;   // the grid's second dimension
        const double us = (double)((wgs + 255) / 256) *
                          (0.5 + (double)((p.KB * wn + 7) / 8) * (0.2 + 0.25 * mb * nt - 0.1 * mb * (wn - 1)));
        if (least == 0. || us < least) least = us, best = i;
    }
    if (best == 0) launch_w4_shape<F16, 1, 1, 1, GROUP>(p, s);
    else if (best == 1) launch_w4_shape<F16, 1, 2, 1, GROUP>(p, s);
    else if (best == 2) launch_w4_shape<F16, 2, 2, 1, GROUP>(p, s);
    else if (best == 3) launch_w4_shape<F16, 3, 2, 1, GROUP>(p, s);
    else if constexpr (GROUP != 32) {
        if (best == 4) launch_w4_shape<F16, 5, 2, 1, GROUP>(p, s);
        else launch_w4_shape<F16, 5, 2, 2, GROUP>(p, s);
    }
}

template <bool F16>
static void launch_w4_group(const W4Args& p, int group, hipStream_t s) {
    if (group == 32) launch_w4<F16, 32>(p, s);
    else if (group == 64) launch_w4<F16, 64>(p, s);
    else launch_w4<F16, 128>(p, s);
}

}  // namespace sfk

extern "C" size_t sf_w4_bytes(int32_t N, int32_t K, int32_t group) {
    if (!sfk::w4_shape_ok(N, K, group)) return 0;
    const size_t n16 = ((size_t)N + 15) / 16;
    return n16 * sfk::w4_kb(K) * 1024 + n16 * sfk::w4_groups(K, group) * 64;
}

extern "C" int sf_w4_pack(const sf_w4_pack_desc* desc, void* out, void* stream) {
    if (!desc || !sfk::w4_shape_ok(desc->N, desc->K, desc->group)) return SF_EINVAL;
    if (!desc->codes || !desc->scales || !out || (reinterpret_cast<uintptr_t>(out) & 15)) return SF_EINVAL;
    if (desc->ldc < desc->K / 2 || desc->lds < desc->K / desc->group ||
        (desc->zeros && desc->ldz < desc->K / desc->group) || (reinterpret_cast<uintptr_t>(desc->scales) & 1))
        return SF_EINVAL;
    if (desc->scale_dtype != SF_F16 && desc->scale_dtype != SF_BF16) return SF_ENOTSUP;
    const int64_t words = (int64_t)(sf_w4_bytes(desc->N, desc->K, desc->group) / 4);
    const int64_t blocks = (words + 255) / 256;
    if (blocks >= 1 << 24) return SF_ENOTSUP;   // a launch counts its threads in 32 bits
    hipLaunchKernelGGL(sfk::w4_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, static_cast<hipStream_t>(stream),
                       *desc, static_cast<uint32_t*>(out), (int)(((int64_t)desc->N + 15) / 16), sfk::w4_kb(desc->K),
                       sfk::w4_groups(desc->K, desc->group));
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}

extern "C" int sf_gemm_w4(const sf_gemm_w4_desc* desc, void* stream) {
    if (!desc || desc->M < 0 || !sfk::w4_shape_ok(desc->N, desc->K, desc->group)) return SF_EINVAL;
    if (desc->M == 0) return SF_OK;
    if (!desc->A || !desc->W || !desc->C) return SF_EINVAL;
    if (((reinterpret_cast<uintptr_t>(desc->A) | reinterpret_cast<uintptr_t>(desc->W)) & 15) || desc->lda < desc->K ||
        (desc->lda & 7) || desc->ldc < desc->N)
        return SF_EINVAL;
    const uintptr_t calign = desc->c_dtype == SF_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(desc->C) & calign) || (reinterpret_cast<uintptr_t>(desc->bias) & 3))
        return SF_EINVAL;
    if (desc->a_dtype != SF_F16 && desc->a_dtype != SF_BF16) return SF_ENOTSUP;
    if (desc->scale_dtype != SF_F16 && desc->scale_dtype != SF_BF16) return SF_ENOTSUP;
    if (desc->c_dtype != SF_F32 && desc->c_dtype != SF_F16 && desc->c_dtype != SF_BF16) return SF_ENOTSUP;
    if (desc->act < SF_ACT_NONE || desc->act > SF_ACT_SILU) return SF_ENOTSUP;
    if (desc->accumulate && desc->c_dtype != SF_F32) return SF_ENOTSUP;
    // the grid's second dimension; a launch counts its threads in 32 bits; a workgroup's rows are addressed in 32 bits
    if (desc->M > 1 << 21 || desc->N > 1 << 25 || desc->lda > 1 << 23) return SF_ENOTSUP;
    sfk::W4Args p = {};
    p.a = static_cast<const uint16_t*>(desc->A);
    p.lda = desc->lda;
    p.KB = sfk::w4_kb(desc->K);
    p.groups = sfk::w4_groups(desc->K, desc->group);
    p.n16 = (int)(((int64_t)desc->N + 15) / 16);
    p.w = static_cast<const uint8_t*>(desc->W);
    p.par = reinterpret_cast<const uint32_t*>(p.w + (int64_t)p.n16 * p.KB * 1024);
    p.bias = desc->bias;
    p.c = desc->C;
    p.ldc = desc->ldc;
    p.M = desc->M;
    p.N = desc->N;
    p.K = desc->K;
    p.scale_f16 = desc->scale_dtype == SF_F16;
    p.act = desc->act;
    p.c_kind = desc->c_dtype == SF_BF16 ? 1 : (desc->c_dtype == SF_F16 ? 2 : 0);
    p.accumulate = desc->accumulate != 0;
    p.vec4 = desc->ldc % 4 == 0 && (reinterpret_cast<uintptr_t>(desc->C) & (p.c_kind == 0 ? 15 : 7)) == 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (desc->a_dtype == SF_F16) sfk::launch_w4_group<true>(p, desc->group, s);
    else sfk::launch_w4_group<false>(p, desc->group, s);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
