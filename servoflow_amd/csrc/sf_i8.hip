// Products in 8-bit integers with a scale for each token and each output channel (gfx950).
//
// C[m][n] = act(s_m t_n sum_k a[m][k] w[n][k] + bias[n]); the sum is exact in 32
// bits.  Activations come as codes, or are quantised first: s_m = max |x_m| / 127,
// a = x / s_m to the nearest, ties to even, exactly -- the quotient by a
// reciprocal, then put right by the sign of what is left of x.
//
// A workgroup of eight waves takes 64 MI x 128 NI outputs, 2 x 4 waves of MI x NI
// tiles of v_mfma_i32_32x32x32_i8.  128 inputs of both operands at a time go
// straight from memory into LDS, rows of 128 bytes whose pieces of 16 are placed by the
// row (piece c of row r at c ^ (r / 2 & 7)), so that the 16 rows that a read of 16 bytes
// takes at a time lie in different banks.  The next 128 inputs are on their way while
// these are multiplied.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>

#include "sf_act.h"
#include "sf_device.h"
#include "sf_hip.h"

namespace sfk {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// ---------------------------------------------------------------- quantising

// Code of x for a step s > 0: |x| <= 127 s but for the step's own rounding.
__device__ __forceinline__ int i8_code(float x, float s, float inv) {
    float q = rintf(x * inv);                      // off by one at most, and only next to a border
    const float r = __builtin_fmaf(-q, s, x);      // exact there: |r| <= s in steps of half an ulp of s
    const float half = 0.5f * s;
    const bool odd = ((int)q & 1) != 0;
    if (r > half || (r == half && odd)) q += 1.f;
    if (r < -half || (r == -half && odd)) q -= 1.f;
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}

template <int KIND>   // 0 fp32, 1 bf16, 2 fp16
__device__ __forceinline__ void i8_load8(const void* row, int k, float (&x)[8]) {
    if (KIND == 0) {
        const f32x4* src = reinterpret_cast<const f32x4*>(static_cast<const float*>(row) + k);
        const f32x4 a = src[0], b = src[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = a[e], x[4 + e] = b[e];
    } else {
        const u32x4 v = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(row) + k);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = v[e >> 1];
            if (KIND == 1) x[e] = __uint_as_float(e & 1 ? h & 0xffff0000u : h << 16);
            else x[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(h >> (16 * (e & 1))));
        }
    }
}

// One workgroup a row.  Up to 8192 inputs stay in registers between the maximum and the codes.
template <int KIND>
__global__ __launch_bounds__(256) void quant_i8_kernel(const void* a, int64_t lda, int K, int8_t* codes, int64_t ldc, float* scale) {
    constexpr int kHeld = 4;
    __shared__ float part[4];
    const int64_t m = blockIdx.x;
    const void* row = static_cast<const char*>(a) + m * lda * (KIND == 0 ? 4 : 2);
    float x[kHeld][8], big = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int k = 8 * (int)threadIdx.x + 2048 * i;
        if (k < K) i8_load8<KIND>(row, k, x[i]);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(x[i][e])), bad = bad || x[i][e] != x[i][e];
    }
    for (int k = 8 * (int)threadIdx.x + 2048 * kHeld; k < K; k += 2048) {
        float y[8];
        i8_load8<KIND>(row, k, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = fmaxf(big, fabsf(y[e])), bad = bad || y[e] != y[e];
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) big = fmaxf(big, __shfl_xor(big, d, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = big;
    bad = __syncthreads_or(bad);
    big = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const float s = bad ? NAN : big / 127.f;   // an infinity: an infinite step, whose products are NaN
    const bool plain = s > 0.f && s < INFINITY;
    const float up = s < 0x1p-60f ? 0x1p100f : 1.f;   // steps whose half or reciprocal is no normal number
    const float step = s * up, inv = 1.f / step;
    if (threadIdx.x == 0) scale[m] = s;
    int8_t* dst = codes + m * ldc;
    auto store = [&](int k, const float (&y)[8]) {
        uint32_t u[2] = {0u, 0u};
        if (plain) {
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e >> 2] |= ((uint32_t)i8_code(y[e] * up, step, inv) & 0xffu) << (8 * (e & 3));
        }
        *reinterpret_cast<uint2*>(dst + k) = uint2{u[0], u[1]};
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int k = 8 * (int)threadIdx.x + 2048 * i;
        if (k < K) store(k, x[i]);
    }
    for (int k = 8 * (int)threadIdx.x + 2048 * kHeld; k < K; k += 2048) {
        float y[8];
        i8_load8<KIND>(row, k, y);
        store(k, y);
    }
}

// ------------------------------------------------------------------ products

struct I8Args {
    const int8_t *a, *w;
    int64_t lda, ldw;
    const float *a_scale, *w_scale, *bias;
    void* c;
    int64_t ldc;
    int M, N, K;
    int act, c_kind, accumulate, vec4;
    int mt, nt;   // tiles
};

// Four columns of a row of C, from column n.
__device__ __forceinline__ void i8_store(const I8Args& p, int m, int n, i32x4 acc) {
    if (m >= p.M || n >= p.N) return;
    const float s = p.a_scale[m];
    const int64_t at = (int64_t)m * p.ldc + n;
    const int cols = min(4, p.N - n);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = i < cols ? apply_act(p.act, (float)acc[i] * s * p.w_scale[n + i] + (p.bias ? p.bias[n + i] : 0.f)) : 0.f;
    if (cols == 4 && p.vec4) {
        if (p.c_kind == 0) {
            f32x4* c = reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + at);
            f32x4 y = {v[0], v[1], v[2], v[3]};
            if (p.accumulate) y += *c;
            *c = y;
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

// Workgroup -> tile.  Workgroups go round the eight XCDs; each XCD takes consecutive tiles, four columns of tiles
// at a time, so that the 32 of its CUs share operands in its L2.
__device__ __forceinline__ void i8_tile(const I8Args& p, int& tm, int& tn) {
    const int all = p.mt * p.nt, xcd = blockIdx.x & 7, per = all >> 3, more = all & 7;
    const int id = xcd * per + min(xcd, more) + (blockIdx.x >> 3);
    const int band = id / (4 * p.mt), in = id % (4 * p.mt), wide = min(4, p.nt - 4 * band);
    tm = in / wide;
    tn = 4 * band + in % wide;
}

template <int MI, int NI>
__global__ __launch_bounds__(512) void gemm_i8_kernel(const I8Args p) {
    constexpr int BM = 64 * MI, BN = 128 * NI, kStage = (BM + BN) * 128;
    __shared__ __attribute__((aligned(1024))) int8_t lds[2 * kStage];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 2, wn = wave & 3, col = lane & 31, g = lane >> 5;
    int tm, tn;
    i8_tile(p, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int rows = min(BM, p.M - m0), cols = min(BN, p.N - n0);
    const __amdgpu_buffer_rsrc_t ars = make_rsrc(p.a + (int64_t)m0 * p.lda, (uint32_t)((rows - 1) * (int)p.lda + p.K));
    const __amdgpu_buffer_rsrc_t wrs = make_rsrc(p.w + (int64_t)n0 * p.ldw, (uint32_t)((cols - 1) * (int)p.ldw + p.K));
    // An instruction brings 8 rows of 128 bytes: lane l the place l & 7 of row l >> 3.
    const int row = lane >> 3, place = lane & 7;
    auto fetch = [&](int k0, int8_t* to) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < (BM + BN) / 64; ++i) {
            const int r8 = 8 * (8 * i + wave);   // of the stage; BM is a multiple of 64
            const bool is_a = i < BM / 64;
            const int r = (is_a ? r8 : r8 - BM) + row;
            const int k = k0 + 16 * (place ^ (r >> 1 & 7));
            const int limit = is_a ? rows : cols;
            const uint32_t at = r < limit && k < p.K ? (uint32_t)r * (uint32_t)(is_a ? p.lda : p.ldw) + (uint32_t)k : 0x80000000u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(is_a ? ars : wrs, (__attribute__((address_space(3))) void*)(to + 128 * r8), 16,
                                                     at, 0, 0, 0);
        }
    };
    i32x16 acc[NI][MI];
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0;
    fetch(0, lds);
    const int steps = (p.K + 127) / 128;
    for (int s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        const int8_t* from = lds + (s & 1) * kStage;
        if (s + 1 < steps) fetch(128 * (s + 1), lds + (1 - (s & 1)) * kStage);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            i32x4 x[MI], w[NI];
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int r = 32 * (MI * wm + i) + col;
                x[i] = *reinterpret_cast<const i32x4*>(from + 128 * r + 16 * ((2 * kk + g) ^ (r >> 1 & 7)));
            }
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int r = 32 * (NI * wn + j) + col;
                w[j] = *reinterpret_cast<const i32x4*>(from + 128 * (BM + r) + 16 * ((2 * kk + g) ^ (r >> 1 & 7)));
            }
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int i = 0; i < MI; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[j], x[i], acc[j][i], 0, 0, 0);
        }
    }
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                i8_store(p, m0 + 32 * (MI * wm + i) + col, n0 + 32 * (NI * wn + j) + 8 * q + 4 * g,
                         i32x4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]});
}

template <int MI, int NI>
static void launch_i8(I8Args p, hipStream_t s) {
    p.mt = (p.M + 64 * MI - 1) / (64 * MI);
    p.nt = (p.N + 128 * NI - 1) / (128 * NI);
    hipLaunchKernelGGL((gemm_i8_kernel<MI, NI>), dim3((unsigned)(p.mt * p.nt)), dim3(512), 0, s, p);
}

static void launch_gemm_i8(const I8Args& p, hipStream_t s) {
    if (p.M <= 64) launch_i8<1, 1>(p, s);
    else launch_i8<4, 2>(p, s);
}

static int quant_i8(const void* a, int64_t lda, int dtype, int M, int K, int8_t* codes, int64_t ldc, float* scale, hipStream_t s) {
    const dim3 grid((unsigned)M), block(256);
    if (dtype == SF_F32) hipLaunchKernelGGL(quant_i8_kernel<0>, grid, block, 0, s, a, lda, K, codes, ldc, scale);
    else if (dtype == SF_BF16) hipLaunchKernelGGL(quant_i8_kernel<1>, grid, block, 0, s, a, lda, K, codes, ldc, scale);
    else hipLaunchKernelGGL(quant_i8_kernel<2>, grid, block, 0, s, a, lda, K, codes, ldc, scale);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}

static inline bool i8_float(int dtype) { return dtype == SF_F32 || dtype == SF_BF16 || dtype == SF_F16; }
static inline bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Rows, inputs and strides that the kernels' 32-bit offsets take: 256 rows of a tile below 2^31 bytes.
constexpr int kI8MaxRows = 1 << 22, kI8MaxInputs = 1 << 16;
constexpr int64_t kI8MaxStride = 1 << 22;

static size_t i8_scales_at(const sf_gemm_i8_desc* d) { return ((size_t)d->M * (size_t)d->K + 15) / 16 * 16; }

}  // namespace sfk

extern "C" int sf_quant_i8(const void* x, int64_t ldx, int32_t dtype, int32_t rows, int32_t cols, int8_t* codes, int64_t ldc,
                           float* scale, void* stream) {
    if (rows < 0 || cols <= 0 || cols % 16) return SF_EINVAL;
    if (!sfk::i8_float(dtype) || rows > sfk::kI8MaxRows || cols > sfk::kI8MaxInputs) return SF_ENOTSUP;
    if (rows == 0) return SF_OK;
    if (!x || !codes || !scale || !sfk::aligned(x, 16) || !sfk::aligned(codes, 8) || !sfk::aligned(scale, 4) || ldx < cols ||
        (ldx & (dtype == SF_F32 ? 3 : 7)) || ldc < cols || (ldc & 7))
        return SF_EINVAL;
    return sfk::quant_i8(x, ldx, dtype, rows, cols, codes, ldc, scale, static_cast<hipStream_t>(stream));
}

extern "C" size_t sf_gemm_i8_workspace_bytes(const sf_gemm_i8_desc* d) {
    if (!d || d->M <= 0 || d->K <= 0 || d->a_dtype == SF_I8) return 0;
    return sfk::i8_scales_at(d) + (size_t)d->M * sizeof(float);
}

extern "C" int sf_gemm_i8(const sf_gemm_i8_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    if (!d || d->M < 0 || d->N <= 0 || d->K <= 0 || d->K % 16) return SF_EINVAL;
    const bool codes = d->a_dtype == SF_I8;
    if (!codes && !sfk::i8_float(d->a_dtype)) return SF_ENOTSUP;
    if (!sfk::i8_float(d->c_dtype) || d->act < SF_ACT_NONE || d->act > SF_ACT_SILU) return SF_ENOTSUP;
    if (d->accumulate && d->c_dtype != SF_F32) return SF_ENOTSUP;
    if (d->M > sfk::kI8MaxRows || d->N > 1 << 25 || d->K > sfk::kI8MaxInputs || d->lda > sfk::kI8MaxStride ||
        d->ldw > sfk::kI8MaxStride || ((int64_t)(d->M + 63) / 64) * ((d->N + 127) / 128) >= 1 << 22)
        return SF_ENOTSUP;
    if (d->M == 0) return SF_OK;
    if (!d->A || !d->W || !d->w_scale || !d->C || (codes && !d->a_scale)) return SF_EINVAL;
    if (!sfk::aligned(d->A, 16) || !sfk::aligned(d->W, 16) || !sfk::aligned(d->a_scale, 4) || !sfk::aligned(d->w_scale, 4) ||
        !sfk::aligned(d->bias, 4) || !sfk::aligned(d->C, d->c_dtype == SF_F32 ? 4 : 2))
        return SF_EINVAL;
    if (d->lda < d->K || (d->lda & (codes ? 15 : d->a_dtype == SF_F32 ? 3 : 7)) || d->ldw < d->K || (d->ldw & 15) || d->ldc < d->N)
        return SF_EINVAL;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    sfk::I8Args p = {};
    p.a = static_cast<const int8_t*>(d->A);
    p.lda = d->lda;
    p.a_scale = d->a_scale;
    if (!codes) {
        if (!workspace || workspace_bytes < sf_gemm_i8_workspace_bytes(d)) return SF_EWORKSPACE;
        if (!sfk::aligned(workspace, 16)) return SF_EINVAL;
        int8_t* held = static_cast<int8_t*>(workspace);
        float* scale = reinterpret_cast<float*>(held + sfk::i8_scales_at(d));
        const int st = sfk::quant_i8(d->A, d->lda, d->a_dtype, d->M, d->K, held, d->K, scale, s);
        if (st != SF_OK) return st;
        p.a = held;
        p.lda = d->K;
        p.a_scale = scale;
    }
    p.w = static_cast<const int8_t*>(d->W);
    p.ldw = d->ldw;
    p.w_scale = d->w_scale;
    p.bias = d->bias;
    p.c = d->C;
    p.ldc = d->ldc;
    p.M = d->M;
    p.N = d->N;
    p.K = d->K;
    p.act = d->act;
    p.c_kind = d->c_dtype == SF_BF16 ? 1 : (d->c_dtype == SF_F16 ? 2 : 0);
    p.accumulate = d->accumulate != 0;
    p.vec4 = d->ldc % 4 == 0 && sfk::aligned(d->C, p.c_kind == 0 ? 16 : 8);
    sfk::launch_gemm_i8(p, s);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
