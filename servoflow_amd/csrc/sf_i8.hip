// Products in 8-bit integers with a scale for each token and each output channel (gfx950).
//
// C[m][n] = act(s_m t_n sum_k a[m][k] w[n][k] + bias[n]); the sum is exact in 32
// bits.  Activations come as codes, or are quantised first: s_m = max |x_m| / 127,
// a = x / s_m to the nearest, ties to even, exactly -- the quotient by a
// reciprocal, then put right by the sign of what is left of x.
//
// Many rows: a workgroup multiplies tiles of v_mfma_i32_32x32x32_i8 from LDS, 128
// inputs of both operands at a time, which come straight from memory.  A row's 128 bytes
// lie there in pieces of 16, piece c of row r at c ^ (r / 2 & 7): the 16 rows that a
// read of 16 bytes takes at a time then lie in different banks.  Few rows: see
// gemm_i8_rows_kernel.
//
// What bounds them (us): 4374 x 8192 x 8192 takes 281 to 290, 2.0 to 2.1 POP/s, where the loads into
// LDS alone take 208, the products with their reads from LDS alone 219 to 227, and a
// large library product of 8-bit integers runs at 2.4 POP/s (292 for this one); with its
// quantising, one pass over 72 MB in and 36 out, 296.  67 x 6144 x 2048 takes 10.4
// with it, 7.8 without: a chain of launch, first operands, stages, join and stores.  1 x 8192
// x 8192 takes 15.0 from memory, 4.5 TB/s of weights.
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

constexpr int kI8MaxInputs = 1 << 16;

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

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Eight inputs of a row.  KIND: 0 fp32, 1 bf16, 2 fp16.
template <int KIND>
struct I8Piece {
    u32x4 v[KIND == 0 ? 2 : 1];
    __device__ __forceinline__ void load(const void* row, int k) {
        const u32x4* from = reinterpret_cast<const u32x4*>(static_cast<const char*>(row) + (int64_t)k * (KIND == 0 ? 4 : 2));
#pragma unroll
        for (int i = 0; i < (KIND == 0 ? 2 : 1); ++i) v[i] = from[i];
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (KIND == 0 ? 2 : 1); ++i) v[i] = u32x4{0, 0, 0, 0};
    }
    // The larger of `most` and these without their signs, as whole numbers: an infinity is above all numbers, and a NaN
    // above that.  16-bit ones two by two.
    __device__ __forceinline__ uint32_t most(uint32_t most) const {
#pragma unroll
        for (int i = 0; i < (KIND == 0 ? 2 : 1); ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (KIND == 0) most = max(most, v[i][e] & 0x7fffffffu);
                else most = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, most),
                                                                                   __builtin_bit_cast(u16x2, v[i][e] & 0x7fff7fffu)));
            }
        return most;
    }
    static __device__ __forceinline__ float value(uint32_t h) {   // of 16 bits
        return KIND == 1 ? __uint_as_float(h << 16) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
    }
    // What `most` found, as the bits of an fp32 number.
    static __device__ __forceinline__ uint32_t bits(uint32_t most) {
        return KIND == 0 ? most : __float_as_uint(value(max(most & 0xffffu, most >> 16)));
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (KIND == 0) x[e] = __uint_as_float(v[e >> 2 & (KIND == 0)][e & 3]);
            else x[e] = value(v[0][e >> 1] >> (16 * (e & 1)) & 0xffffu);
        }
    }
};

// A row's step from the bits of its largest |x|, and the same for i8_code where the step's half or reciprocal is no normal
// number.
struct I8Step {
    float s, step, inv, up;
    bool plain;   // no: codes 0 (a row of zeros; an infinity or a NaN, whose step makes the products NaN)
    __device__ __forceinline__ explicit I8Step(uint32_t big) {
        s = __uint_as_float(big) / 127.f;
        plain = s > 0.f && s < INFINITY;
        up = s < 0x1p-60f ? 0x1p100f : 1.f;
        step = s * up;
        inv = 1.f / step;
    }
    // x times the reciprocal is off by less than 127 2^-23 and a rounding: where it is further than 2e-5 from the middle of two
    // codes the nearer one is right, and one addition of 1.5 2^23 leaves it in the low bits.  False where it is not for one of
    // these eight (for one in 3000), or the step asks for `up`: slow_codes.
    __device__ __forceinline__ bool codes(const float (&y)[8], uint2& u) const {
        constexpr float kWhole = 12582912.f;
        float far = 0.f;
        uint32_t z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float n = __builtin_fmaf(y[e], inv, kWhole);
            far = fmaxf(far, fabsf(__builtin_fmaf(y[e], inv, kWhole - n)));
            z[e] = __float_as_uint(n);
        }
        auto four = [&](int i) {
            return __builtin_amdgcn_perm(z[i + 1], z[i], 0x0c0c0400u) | __builtin_amdgcn_perm(z[i + 3], z[i + 2], 0x04000c0cu);
        };
        u = plain ? uint2{four(0), four(4)} : uint2{0u, 0u};
        return !plain || (up == 1.f && far < 0.49998f);
    }
    __device__ __forceinline__ uint2 slow_codes(const float (&y)[8]) const {
        uint32_t u[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e >> 2] |= ((uint32_t)i8_code(y[e] * up, step, inv) & 0xffu) << (8 * (e & 3));
        return uint2{u[0], u[1]};
    }
};

// One workgroup a row.  Up to 8192 inputs stay in registers between the maximum and the codes.  4374 rows of 8192 bf16
// inputs take 20 us (21 at the rate of a copy; 27 with i8_code for all of them), 67 x 2048 3.3, a launch and a row's chain.
template <int KIND>
__global__ __launch_bounds__(256) void quant_i8_kernel(const void* a, int64_t lda, int K, int8_t* codes, int64_t ldc, float* scale) {
    constexpr int kHeld = 4;
    __shared__ uint32_t part[4];
    const int64_t m = blockIdx.x;
    const void* row = static_cast<const char*>(a) + m * lda * (KIND == 0 ? 4 : 2);
    I8Piece<KIND> x[kHeld];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int k = 8 * (int)threadIdx.x + 2048 * i;
        if (k < K) x[i].load(row, k);
        else x[i].clear();
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = x[i].most(most);
    for (int k = 8 * (int)threadIdx.x + 2048 * kHeld; k < K; k += 2048) {
        I8Piece<KIND> y;
        y.load(row, k);
        most = y.most(most);
    }
    most = I8Piece<KIND>::bits(most);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    const I8Step st(max(max(part[0], part[1]), max(part[2], part[3])));
    if (threadIdx.x == 0) scale[m] = st.s;
    int8_t* dst = codes + m * ldc;
    uint32_t again = 0;   // pieces of the thread, 32 at most
    auto store = [&](int i, int k, const I8Piece<KIND>& piece) {
        float y[8];
        uint2 u;
        piece.floats(y);
        if (!st.codes(y, u)) again |= 1u << i;
        *reinterpret_cast<uint2*>(dst + k) = u;
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int k = 8 * (int)threadIdx.x + 2048 * i;
        if (k < K) store(i, k, x[i]);
    }
    for (int i = kHeld, k = 8 * (int)threadIdx.x + 2048 * kHeld; k < K; ++i, k += 2048) {
        I8Piece<KIND> y;
        y.load(row, k);
        store(i, k, y);
    }
    for (; again; again &= again - 1) {   // from memory once more: few, and the code stays small
        const int k = 8 * (int)threadIdx.x + 2048 * __builtin_ctz(again);
        I8Piece<KIND> piece;
        float y[8];
        piece.load(row, k);
        piece.floats(y);
        *reinterpret_cast<uint2*>(dst + k) = st.slow_codes(y);
    }
}
static_assert(kI8MaxInputs <= 32 * 2048, "a bit for each of a thread's pieces");

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
    const void* x;   // rows to be quantised by the workgroup that multiplies them
    int64_t ldx;
};

// Scales and bias of four columns from n on (0 behind the last).
struct I8Columns {
    f32x4 scale, bias;
};
__device__ __forceinline__ I8Columns i8_columns(const I8Args& p, int n) {
    I8Columns c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = n + i < p.N;
        c.scale[i] = in ? p.w_scale[n + i] : 0.f;
        c.bias[i] = in && p.bias ? p.bias[n + i] : 0.f;
    }
    return c;
}

// Four columns of a row of C, from column n.
__device__ __forceinline__ void i8_store(const I8Args& p, int m, int n, i32x4 acc, float s, const I8Columns& c4) {
    if (m >= p.M || n >= p.N) return;
    const int64_t at = (int64_t)m * p.ldc + n;
    const int cols = min(4, p.N - n);
    float v[4];
    // acc is 2^30 at most: beside a step of 2^96 and more 2^30 of it goes to the other scale, or a sum times the step alone could be
    // beyond fp32.
    const float up = s >= 0x1p96f ? 0x1p30f : 1.f, low = s >= 0x1p96f ? s * 0x1p-30f : s;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)acc[i] * low * (c4.scale[i] * up) + c4.bias[i];
    if (p.act) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = apply_act(p.act, v[i]);
    }
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

// WM x WN waves of MI x NI tiles each.  128 inputs of both operands are a stage, whole lines of memory (with stages of 64
// inputs, two to a line, the loads alone took 217 us of 4096 x 8192 x 8192, so 166); STAGES of them in a ring.  A quarter's
// operands are read under the products of the one before it, those of the next stage's first under the last one's,
// behind the one barrier of a stage.
// KS groups of waves deal the stages, each with a ring of its own, and join in LDS.
template <int MI, int NI, int WM, int WN, int STAGES, int KS = 1>
__global__ __launch_bounds__(64 * WM * WN * KS) void gemm_i8_kernel(const I8Args p) {
    constexpr int BM = 32 * MI * WM, BN = 32 * NI * WN, NW = WM * WN, kStage = (BM + BN) * 128;   // NW: of a group
    constexpr int kLoads = (BM + BN) / 8 / NW;   // instructions of a wave, 8 rows each
    static_assert(BM % 8 == 0 && kLoads * 8 * NW == BM + BN, "whole instructions");
    // One array: beside a second one the compiler waits for every load into LDS before each read from it.
    __shared__ __attribute__((aligned(1024))) int8_t lds[KS * STAGES * kStage + 4 * (BM + 2 * BN)];
    const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = all_waves / NW, wave = all_waves % NW;
    const int wm = wave / WN, wn = wave % WN, col = lane & 31, g = lane >> 5;
    int8_t* const ring = lds + group * STAGES * kStage;
    int tm, tn;
    i8_tile(p, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    const int rows = min(BM, p.M - m0), cols = min(BN, p.N - n0);
    // Scales and bias wait in LDS: read from memory tile by tile at the end they cost 25 us of a 256 x 256 tile.
    float* w_scale = reinterpret_cast<float*>(lds + KS * STAGES * kStage);
    float* bias = w_scale + BN;
    float* a_scale = bias + BN;
    static_assert(BM <= 64 * NW * KS && BN <= 64 * NW * KS, "a thread for each");
    if ((int)threadIdx.x < BM) a_scale[threadIdx.x] = (int)threadIdx.x < rows ? p.a_scale[m0 + threadIdx.x] : 0.f;
    if ((int)threadIdx.x < BN) {
        const bool in = (int)threadIdx.x < cols;
        w_scale[threadIdx.x] = in ? p.w_scale[n0 + threadIdx.x] : 0.f;
        bias[threadIdx.x] = in && p.bias ? p.bias[n0 + threadIdx.x] : 0.f;
    }
    const __amdgpu_buffer_rsrc_t ars = make_rsrc(p.a + (int64_t)m0 * p.lda, (uint32_t)((rows - 1) * (int)p.lda + p.K));
    const __amdgpu_buffer_rsrc_t wrs = make_rsrc(p.w + (int64_t)n0 * p.ldw, (uint32_t)((cols - 1) * (int)p.ldw + p.K));
    // Lane l brings the place l & 7 of row l >> 3: of row r the inputs 16 (place ^ (r / 2 & 7)).  Rows behind the last, and
    // inputs behind K, are behind the buffer's end and come as zeros.
    uint32_t at[kLoads];
    int k_lane[2];   // of rows 0 .. 7 and 8 .. 15 of 16
#pragma unroll
    for (int i = 0; i < 2; ++i) k_lane[i] = 16 * ((lane & 7) ^ (4 * i + (lane >> 4)));
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int piece = i * NW + wave;
        const bool is_a = piece < BM / 8;
        const int r = 8 * (is_a ? piece : piece - BM / 8) + (lane >> 3);
        at[i] = r < (is_a ? rows : cols) ? (uint32_t)r * (uint32_t)(is_a ? p.lda : p.ldw) + (uint32_t)k_lane[piece & 1] : 0x80000000u;
    }
    auto fetch = [&](int s, int8_t* to) __attribute__((always_inline)) {
        const int k0 = 128 * (KS * s + group);
        auto load = [&](int i, uint32_t off) __attribute__((always_inline)) {
            const int piece = i * NW + wave;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(piece < BM / 8 ? ars : wrs,
                                                     (__attribute__((address_space(3))) void*)(to + 1024 * piece), 16, off, 0, 0, 0);
        };
        if (k0 + 128 <= p.K) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) load(i, at[i] + (uint32_t)k0);   // behind the end stays there: k0 is below 2^18
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                load(i, k0 + k_lane[(i * NW + wave) & 1] < p.K ? at[i] + (uint32_t)k0 : 0x80000000u);
        }
    };
    i32x16 acc[NI][MI];
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[j][i][e] = 0;
    i32x4 x[2][MI], w[2][NI];
    // Quarter kk of a stage: lane (col, g) holds piece 2 kk + g of its row.
    auto operands = [&](const int8_t* from, int kk) __attribute__((always_inline)) {
        auto read = [&](int r0) __attribute__((always_inline)) {
            const int r = r0 + col;
            return *reinterpret_cast<const i32x4*>(from + 128 * r + 16 * ((2 * kk + g) ^ (r >> 1 & 7)));
        };
#pragma unroll
        for (int j = 0; j < NI; ++j) w[kk & 1][j] = read(BM + 32 * (NI * wn + j));
#pragma unroll
        for (int i = 0; i < MI; ++i) x[kk & 1][i] = read(32 * (MI * wm + i));
    };
    auto multiply = [&](int kk) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[kk & 1][j], x[kk & 1][i], acc[j][i], 0, 0, 0);
    };
    // What the wave has read is in registers and its loads of the stage that follows are in LDS; so it is of every wave behind
    // the barrier.
    auto meet = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((STAGES - 2) * kLoads) : "memory");
        if (NW > 1) __builtin_amdgcn_s_barrier();   // a wave alone has its ring to itself
        asm volatile("" ::: "memory");
    };
    const int steps = (p.K + 128 * KS - 1) / (128 * KS);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) fetch(i, ring + i * kStage);   // behind K: zeros
    if (NW == 1) __syncthreads();   // the scales
    meet();
    int here = 0, last = (STAGES - 1) * kStage;   // the stage that is multiplied, and the place of the one before it
    operands(ring, 0);
    for (int s = 0; s < steps; ++s) {
        fetch(s + STAGES - 1, ring + last);   // every wave has read what is there
        operands(ring + here, 1);
        multiply(0);
        operands(ring + here, 2);
        multiply(1);
        operands(ring + here, 3);
        multiply(2);
        meet();
        last = here;
        here = here == (STAGES - 1) * kStage ? 0 : here + kStage;
        operands(ring + here, 0);   // behind the last stage: not used
        multiply(3);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing comes into LDS behind the end
    // The groups' sums: each stores the quarters q = group, group + KS, ... of every tile.
    constexpr int kTiles = MI * NI * 4;
    static_assert(KS == 1 || (4 % KS == 0 && NW * kTiles * 1024 <= STAGES * kStage), "the join takes the rings' place");
    i32x4* sums = reinterpret_cast<i32x4*>(lds) + (KS * wave * kTiles + group) * 64 + lane;   // [wave][quarter of a tile][group][lane]
    if constexpr (KS > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    sums[((j * MI + i) * 4 + q) * KS * 64] = i32x4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
        __syncthreads();
        sums -= group * 64;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int m = 32 * (MI * wm + i) + col;
        const float sm = a_scale[m];
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int of = 0; of < 4 / KS; ++of) {
                const int q = KS * of + (KS > 1 ? group : 0);
                const int n = 32 * (NI * wn + j) + 8 * q + 4 * g;
                i32x4 v;
                if constexpr (KS > 1) {
                    v = sums[((j * MI + i) * 4 + q) * KS * 64];
#pragma unroll
                    for (int k = 1; k < KS; ++k) v += sums[(((j * MI + i) * 4 + q) * KS + k) * 64];
                } else {
                    v = i32x4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
                }
                const I8Columns c = {*reinterpret_cast<const f32x4*>(w_scale + n), *reinterpret_cast<const f32x4*>(bias + n)};
                i8_store(p, m0 + m, n0 + n, v, sm, c);
            }
    }
}

// Few rows: MB tiles of 16 rows against NT tiles of 16 columns to a workgroup, whose eight waves deal the inputs, 128 at a
// time, and join in LDS.  Both operands go straight into registers, DEPTH blocks of inputs ahead; the weights are read once.
// KIND: of rows that the workgroup quantises itself (as I8Piece takes it; MB 1), -1 for codes.  Up to kFusedCodes inputs in all:
// every workgroup does it for itself, while its weights are on their way, and a launch is saved.
constexpr int kFusedCodes = 8192;
template <int MB, int NT, int DEPTH, int KIND = -1>
__global__ __launch_bounds__(512) void gemm_i8_rows_kernel(const I8Args p) {
    constexpr int NW = 8;
    __shared__ i32x4 sums[NW][MB * NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int n0 = 16 * NT * blockIdx.x, m0 = 16 * MB * blockIdx.y;
    const int rows = min(16 * MB, p.M - m0), cols = min(16 * NT, p.N - n0);
    constexpr bool kFused = KIND >= 0;
    __shared__ __attribute__((aligned(16))) int8_t held[kFused ? kFusedCodes + 16 * 16 + 128 : 16];   // rows 16 bytes further apart than K
    __shared__ uint32_t biggest[16];
    const __amdgpu_buffer_rsrc_t ars = make_rsrc(p.a + (int64_t)m0 * p.lda, kFused ? 0u : (uint32_t)((rows - 1) * (int)p.lda + p.K));
    const __amdgpu_buffer_rsrc_t wrs = make_rsrc(p.w + (int64_t)n0 * p.ldw, (uint32_t)((cols - 1) * (int)p.ldw + p.K));
    uint32_t wat[NT], xat[MB];   // rows behind the last repeat it; they are not stored
#pragma unroll
    for (int t = 0; t < NT; ++t) wat[t] = (uint32_t)min(16 * t + r, cols - 1) * (uint32_t)p.ldw;
#pragma unroll
    for (int b = 0; b < MB; ++b) xat[b] = (uint32_t)min(16 * b + r, rows - 1) * (uint32_t)(kFused ? p.K + 16 : p.lda);
    constexpr int kUnits = (NT * MB + NW - 1) / NW;   // tiles that a wave joins and stores
    float sm[kUnits];
    I8Columns cn[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = wave + i * NW, m = m0 + 16 * (u % MB) + r;
        if (u >= NT * MB) break;
        sm[i] = !kFused && m < p.M ? p.a_scale[m] : 0.f;
        cn[i] = i8_columns(p, n0 + 16 * (u / MB) + 4 * g);
    }
    i32x4 acc[NT][MB];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = i32x4{0, 0, 0, 0};
    i32x4 w[DEPTH][NT][2], x[DEPTH][MB][2];
    auto load = [&](int d, int kb) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t k = 128u * kb + 64u * j + 16u * g;
            const bool in = (int)k < p.K;   // behind K: zeros
#pragma unroll
            for (int t = 0; t < NT; ++t) w[d][t][j] = __builtin_bit_cast(i32x4, buffer_load16(wrs, in ? wat[t] + k : 0x80000000u));
#pragma unroll
            for (int b = 0; b < MB && !kFused; ++b) x[d][b][j] = __builtin_bit_cast(i32x4, buffer_load16(ars, in ? xat[b] + k : 0x80000000u));
        }
    };
    const int blocks = (p.K + 127) / 128;
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
        if (wave + d * NW < blocks) load(d, wave + d * NW);
    if constexpr (kFused) {
        constexpr int kChunks = kFusedCodes / 8 / 512;   // of 8 inputs, of a thread
        const int per_row = p.K / 8, all = p.M * per_row;
        I8Piece<KIND> y[kChunks];
        int at[kChunks];
        if (threadIdx.x < 16) biggest[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            const int c = (int)threadIdx.x + 512 * i, row = c / per_row;
            at[i] = c < all ? row : -1;
            if (c < all) y[i].load(static_cast<const char*>(p.x) + row * p.ldx * (KIND == 0 ? 4 : 2), 8 * (c % per_row));
        }
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
            if (at[i] >= 0) atomicMax(&biggest[at[i]], I8Piece<KIND>::bits(y[i].most(0u)));
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            if (at[i] < 0) continue;
            const int c = (int)threadIdx.x + 512 * i;
            const I8Step st(biggest[at[i]]);
            float x8[8];
            uint2 u;
            y[i].floats(x8);
            if (!st.codes(x8, u)) u = st.slow_codes(x8);
            *reinterpret_cast<uint2*>(held + at[i] * (p.K + 16) + 8 * (c % per_row)) = u;
        }
#pragma unroll
        for (int i = 0; i < kUnits; ++i) sm[i] = I8Step(biggest[r]).s;   // rows behind the last: 0, not stored
        __syncthreads();
    }
    for (int kb = wave; kb < blocks; kb += DEPTH * NW) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (kb + d * NW >= blocks) break;
            if constexpr (kFused) {   // behind K anything, against weights of 0
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    x[d][0][j] = *reinterpret_cast<const i32x4*>(held + xat[0] + 128 * (kb + d * NW) + 64 * j + 16 * g);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int b = 0; b < MB; ++b) acc[t][b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d][t][j], x[d][b][j], acc[t][b], 0, 0, 0);
            if (kb + (d + DEPTH) * NW < blocks) load(d, kb + (d + DEPTH) * NW);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) sums[wave][t * MB + b][lane] = acc[t][b];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = wave + i * NW;
        if (u >= NT * MB) break;
        i32x4 v = sums[0][u][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += sums[w][u][lane];
        i8_store(p, m0 + 16 * (u % MB) + r, n0 + 16 * (u / MB) + 4 * g, v, sm[i], cn[i]);
    }
}

template <int MI, int NI, int WM, int WN, int STAGES, int KS = 1>
static void launch_i8(I8Args p, hipStream_t s) {
    p.mt = (p.M + 32 * MI * WM - 1) / (32 * MI * WM);
    p.nt = (p.N + 32 * NI * WN - 1) / (32 * NI * WN);
    hipLaunchKernelGGL((gemm_i8_kernel<MI, NI, WM, WN, STAGES, KS>), dim3((unsigned)(p.mt * p.nt)), dim3(64 * WM * WN * KS), 0, s, p);
}

template <int MB, int NT, int DEPTH>
static void launch_i8_rows(const I8Args& p, hipStream_t s) {
    const dim3 grid((unsigned)((p.N + 16 * NT - 1) / (16 * NT)), (unsigned)((p.M + 16 * MB - 1) / (16 * MB)));
    hipLaunchKernelGGL((gemm_i8_rows_kernel<MB, NT, DEPTH>), grid, dim3(512), 0, s, p);
}

// The shape whose estimate is the smallest.  A CU takes its share of the workgroups, `resident` at a time; such a round
// of k of them takes `each` us and for every step max(alone, shared k): a workgroup's own chain, or what the CU fetches
// and multiplies.  A step is 128 inputs of a tile for each group of waves, 1024 of the forms for few rows (a block for each
// wave).  Fitted to 585 products of 1..4374 rows, 256..8192 columns and 512..8192 inputs, where the choice costs 1% in the
// mean, and up to 29%, over the fastest of 21 shapes, with weights that mostly come from the memory-side cache; from memory
// the tiles of 32 rows lose a third where one slab of them reads all weights (1 x 2048 x 8192: 10.3, with 16 x 16 7.6).  us:
//   1 x 8192 x 8192 14.0 with 16 x 16, 16.5 with 16 x 32 (weights from memory); 67 x 2048 x 8192 8.3 with 32 x 32 in four
//   groups, 17.0 with 64 x 64 in one; 134 x 2048 x 8192 11.3 with 32 x 64 in four, 14.1 with 64 x 64 in two, 18.7 in one;
//   536 x 1000 x 8192 14.8 with 64 x 64 in two, 19.0 in one, 21.7 with 32 x 64 in four; 268 x 8192 x 8192 35.3 with
//   128 x 128 and 16 waves, 37.0 with 8; 4374 x 2048 x 2048 29.5 with 192 x 256, 36.5 with 128 x 128; 4374 x 8192 x 8192
//   290 with 192 x 256 (three full rounds of workgroups), 346 with 256 x 256.
struct I8Shape {
    int bm, bn, step, resident;
    double start, alone, shared, each;
};
constexpr I8Shape kI8Shapes[] = {
    {16, 16, 1024, 4, 1.91, 0.0, 0.877, 0.05}, {16, 32, 1024, 4, 1.90, 0.0, 1.337, 0.0},  {32, 32, 512, 1, 1.28, 0.328, 0.0, 2.15},
    {32, 32, 512, 2, 1.05, 0.468, 0.335, 1.97}, {32, 64, 512, 1, 1.05, 0.509, 0.0, 2.37}, {64, 64, 256, 1, 0.99, 0.357, 0.0, 2.67},
    {64, 128, 256, 1, 0.05, 0.520, 0.0, 4.25}, {64, 128, 128, 1, 0.58, 0.312, 0.0, 3.10}, {128, 128, 128, 2, 0.0, 0.594, 0.530, 4.42},
    {128, 128, 128, 1, 0.0, 0.423, 0.0, 4.66}, {128, 256, 128, 1, 0.0, 0.770, 0.0, 7.76}, {192, 256, 128, 1, 0.0, 1.065, 0.0, 9.88},
};

static int i8_shape(const I8Args& p) {
    int best = -1;
    double least = 0.;
    for (int i = 0; i < (int)(sizeof(kI8Shapes) / sizeof(kI8Shapes[0])); ++i) {
        const I8Shape& f = kI8Shapes[i];
        const int64_t slabs = (p.M + f.bm - 1) / f.bm, wgs = slabs * ((p.N + f.bn - 1) / f.bn);
        if ((f.step == 1024 && slabs > 65535) || (wgs >= 1 << 21 && f.bm < 128)) continue;   // a grid's second dimension; its threads
        const int64_t n = (wgs + 255) / 256, steps = (p.K + f.step - 1) / f.step;
        auto round = [&](int64_t k) { return k ? f.each + (double)steps * std::max(f.alone, f.shared * (double)k) : 0.; };
        double us = f.start + (double)(n / f.resident) * round(f.resident) + round(n % f.resident);
        if (f.bm == 32 && slabs == 1) us *= 1.3;
        if (best < 0 || us < least) least = us, best = i;
    }
    return best;
}

// Few inputs are quantised where they are multiplied.  us in a graph, so and in two launches: 1 x 2048 x 2048 4.1 and 5.8,
// 1 x 8192 x 8192 14.2 and 18.9, 5 x 2051 x 1152 4.9 and 6.0, 4 x 8192 x 2048 8.6 and 8.4; of more inputs every workgroup's
// own quantising counts: 8 x 8192 x 2048 took 4 more.
static inline bool i8_fused(const sf_gemm_i8_desc* d) {
    return d->a_dtype != SF_I8 && d->M <= 16 && (int64_t)d->M * d->K <= kFusedCodes;
}
template <int KIND>
static void launch_i8_fused(const I8Args& p, hipStream_t s) {
    const bool narrow = p.N <= 16 * 512;   // as many workgroups as two to a CU, or wider ones
    const dim3 grid((unsigned)(narrow ? (p.N + 15) / 16 : (p.N + 31) / 32));
    if (narrow) hipLaunchKernelGGL((gemm_i8_rows_kernel<1, 1, 4, KIND>), grid, dim3(512), 0, s, p);
    else hipLaunchKernelGGL((gemm_i8_rows_kernel<1, 2, 3, KIND>), grid, dim3(512), 0, s, p);
}

static void launch_gemm_i8(const I8Args& p, hipStream_t s) {
    switch (i8_shape(p)) {
    case 0: return launch_i8_rows<1, 1, 4>(p, s);
    case 1: return launch_i8_rows<1, 2, 3>(p, s);
    case 2: return launch_i8<1, 1, 1, 1, 4, 4>(p, s);
    case 3: return launch_i8<1, 1, 1, 1, 2, 4>(p, s);
    case 4: return launch_i8<1, 1, 1, 2, 3, 4>(p, s);
    case 5: return launch_i8<1, 1, 2, 2, 4, 2>(p, s);
    case 6: return launch_i8<1, 1, 2, 4, 3, 2>(p, s);
    case 7: return launch_i8<1, 1, 2, 4, 4>(p, s);
    case 8: return launch_i8<2, 1, 2, 4, 2>(p, s);
    case 9: return launch_i8<1, 1, 4, 4, 4>(p, s);
    case 10: return launch_i8<2, 2, 2, 4, 3>(p, s);
    default: return launch_i8<3, 2, 2, 4, 2>(p, s);
    }
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
constexpr int kI8MaxRows = 1 << 22;
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
    if (!d || d->M <= 0 || d->K <= 0 || d->a_dtype == SF_I8 || sfk::i8_fused(d)) return 0;
    return sfk::i8_scales_at(d) + (size_t)d->M * sizeof(float);
}

extern "C" int sf_gemm_i8(const sf_gemm_i8_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    if (!d || d->M < 0 || d->N <= 0 || d->K <= 0 || d->K % 16) return SF_EINVAL;
    const bool codes = d->a_dtype == SF_I8;
    if (!codes && !sfk::i8_float(d->a_dtype)) return SF_ENOTSUP;
    if (!sfk::i8_float(d->c_dtype) || d->act < SF_ACT_NONE || d->act > SF_ACT_SILU) return SF_ENOTSUP;
    if (d->accumulate && d->c_dtype != SF_F32) return SF_ENOTSUP;
    if (d->M > sfk::kI8MaxRows || d->N > 1 << 25 || d->K > sfk::kI8MaxInputs || d->lda > sfk::kI8MaxStride ||
        d->ldw > sfk::kI8MaxStride || ((int64_t)(d->M + 63) / 64) * ((d->N + 63) / 64) >= 1 << 22)
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
    const bool fused = sfk::i8_fused(d);
    if (fused) {
        p.x = d->A;
        p.ldx = d->lda;
    } else if (!codes) {
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
    if (!fused) sfk::launch_gemm_i8(p, s);
    else if (d->a_dtype == SF_F32) sfk::launch_i8_fused<0>(p, s);
    else if (d->a_dtype == SF_BF16) sfk::launch_i8_fused<1>(p, s);
    else sfk::launch_i8_fused<2>(p, s);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
