// One token from each row of logits: temperature, top-k, top-p, min-p (gfx950).
//
// With the row's largest logit m a token's weight is 2^43 exp((l - m) / temperature)
// rounded to a whole number, from a table of 2^(j / 128) and four terms of the series
// in 64 bits (1.3e-15 relative).  Sums of weights are sums of whole numbers below
// 2^63 for up to 2^20 tokens: their order does not matter, so a row's token depends
// on the row alone, and neighbours in the running sum differ by far more than it is
// off -- a vocabulary of 131072 in 32 bits would draw another token than 64 bits do
// once in some ten rows.  What is below 2^-44 of the largest counts as nothing.
//
// Every filter keeps a prefix of the tokens in falling order, so all that is ever
// asked of that order is the first position whose running count or running weight
// passes a number.  Nothing is sorted for it: the row is spread over 2048 buckets
// of (l - m) / temperature, 1 / 44.5 octave each, with count and weight of each; the bucket
// that holds the position is found from their running sums, and only its
// tokens (with those above it where they are few) are put in order, in LDS.  A
// bucket of more than 2048 tokens is halved by keys, 2048 parts at a time, until one
// value is left, of which the tokens go by index.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sf_device.h"
#include "sf_hip.h"

namespace sfk {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBuckets = 2 * kSampleThreads;        // two to a thread
constexpr int kSampleList = 2 * kSampleThreads;     // tokens put in order at a time, two to a thread
constexpr int kExpBits = 7;
constexpr float kOctaves = 46.f;                    // 2^-46 and below: no weight
constexpr double kUnit = 8796093022208.;            // 2^43

struct SampleArgs {
    const void* logits;
    int64_t ld;
    const float *u, *temperature, *top_p, *min_p;   // [rows], NULL: the scalars below
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    int32_t top_k1;
    int V;
    int32_t* token;
    float* logprob;
};

struct SampleShared {
    uint64_t mass[kBuckets];     // running, once summed
    uint32_t count[kBuckets];
    uint32_t cursor[kBuckets];   // tokens of a bucket that are in the list; counts of index ranges
    union {
        struct {
            uint64_t raw[kSampleList];      // ~key << 32 | index: falling order of keys, rising of indexes
            uint64_t sorted[kSampleList];
            uint64_t run[kSampleList];      // running weight, from the list's first
        } list;
        struct {
            uint64_t mass[kBuckets];
            uint32_t count[kBuckets];
        } part;
    };
    double exp2[1 << kExpBits];
    uint64_t wave64[kSampleWaves];
    uint32_t wave32[kSampleWaves];
    // what one thread found
    uint32_t found, found_count, found_before;
    uint64_t found_mass, found_mass_before, found_entry;
    uint32_t lo, hi;
    int token;
};

// fp32 -> whole numbers in the same order, and back; -0 counts as 0.
__device__ __forceinline__ uint32_t sample_key(float l) {
    const uint32_t b = __float_as_uint(l + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sample_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// KIND: 0 fp32, 1 bf16, 2 fp16 (as SF_F32, ... map).
template <int KIND>
struct SampleRow {
    static constexpr int E = KIND == 0 ? 4 : 8;   // elements of 16 bytes
    const char* base;
    int V;
    __device__ __forceinline__ float one(int i) const {
        if (KIND == 0) return reinterpret_cast<const float*>(base)[i];
        const uint16_t h = reinterpret_cast<const uint16_t*>(base)[i];
        return KIND == 1 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
    }
    // f(logit, index) for every element, each thread its own: whole pieces of 16 bytes, and singly what lies before the
    // first and behind the last.
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        const int t = threadIdx.x;
        const int size = KIND == 0 ? 4 : 2;
        const int head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / size);
        const int pieces = (V - head) / E, tail = head + pieces * E;
        const u32x4* from = reinterpret_cast<const u32x4*>(base + head * size);
        for (int c0 = t; c0 < pieces; c0 += 4 * kSampleThreads) {
            u32x4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c0 + j * kSampleThreads < pieces) v[j] = from[c0 + j * kSampleThreads];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = c0 + j * kSampleThreads;
                if (c >= pieces) break;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    float l;
                    if (KIND == 0) l = __uint_as_float(v[j][e & 3]);
                    else if (KIND == 1) l = __uint_as_float(e & 1 ? v[j][e >> 1] & 0xffff0000u : v[j][e >> 1] << 16);
                    else l = (float)__builtin_bit_cast(_Float16, (uint16_t)(v[j][e >> 1] >> (16 * (e & 1))));
                    f(l, head + c * E + e);
                }
            }
        }
        if (t < head) f(one(t), t);
        if (t < V - tail) f(one(tail + t), tail + t);
    }
};

// What a logit counts for.
struct SampleScale {
    float m, per_bucket;
    double octaves;                // 128 log2 e / temperature
    __device__ __forceinline__ float below(float l) const { return l == m ? 0.f : l - m; }
    __device__ __forceinline__ int bucket(float l) const {   // kBuckets and more: no weight
        const float b = -below(l) * per_bucket;
        return b < (float)kBuckets ? (int)b : kBuckets;
    }
    __device__ __forceinline__ double exponent(float l) const {   // of two, times 128
        return l == m ? 0. : ((double)l - (double)m) * octaves;
    }
    __device__ __forceinline__ uint64_t weight(double y, const double* table) const {
        const double magic = 6755399441055744.;   // 1.5 2^52: the nearest whole number in the low bits
        const double z = fmax(y, -128. * 64.) + magic;
        const int n = (int)(uint32_t)__double_as_longlong(z);
        const double r = (fmax(y, -128. * 64.) - (z - magic)) * (M_LN2 / 128.);
        const double p = 1. + r * (1. + r * (0.5 + r * (1. / 6. + r * (1. / 24.))));
        const double w = ldexp(p * table[n & 127], (n >> kExpBits) + 43);
        return (uint64_t)__double_as_longlong(w + 4503599627370496.) & 0xfffffffffffffull;   // + 2^52: rounded
    }
};

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
    const uint32_t lo = __shfl_up((uint32_t)v, d, 64), hi = __shfl_up((uint32_t)(v >> 32), d, 64);
    return (uint64_t)hi << 32 | lo;
}

// Running sums over 2048 counts and weights (either may be null), two to a thread.
__device__ __forceinline__ void sample_running(SampleShared& s, uint32_t* count, uint64_t* mass) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t c0 = 0, c = 0;
    uint64_t m0 = 0, m = 0;
    if (count) c0 = count[2 * t], c = c0 + count[2 * t + 1];
    if (mass) m0 = mass[2 * t], m = m0 + mass[2 * t + 1];
    uint32_t ci = c;
    uint64_t mi = m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t a = __shfl_up(ci, d, 64);
        const uint64_t b = shfl_up64(mi, d);
        if (lane >= d) ci += a, mi += b;
    }
    if (lane == 63) s.wave32[wave] = ci, s.wave64[wave] = mi;
    __syncthreads();
    for (int w = 0; w < wave; ++w) ci += s.wave32[w], mi += s.wave64[w];
    if (count) count[2 * t] = ci - c + c0, count[2 * t + 1] = ci;
    if (mass) mass[2 * t] = mi - m + m0, mass[2 * t + 1] = mi;
    __syncthreads();
}

// The first position whose running count reaches `count`, or whose running weight reaches (strict: passes) `mass`.
struct SampleQuery {
    uint32_t count;
    double mass;
    bool strict;
    __device__ __forceinline__ bool at(uint32_t c, uint64_t m) const {
        return c >= count || (strict ? (double)m > mass : (double)m >= mass);
    }
};

// Finds, among 2048 running counts and weights that start from (c0, m0), the first that answers q; s.found and what is
// before it.
__device__ __forceinline__ void sample_find(SampleShared& s, const uint32_t* count, const uint64_t* mass, uint32_t c0, uint64_t m0,
                                            const SampleQuery& q) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = 2 * (int)threadIdx.x + j;
        const uint32_t cb = c0 + (i ? count[i - 1] : 0u);
        const uint64_t mb = m0 + (i ? mass[i - 1] : 0ull);
        if (q.at(c0 + count[i], m0 + mass[i]) && (i == 0 || !q.at(cb, mb))) {
            s.found = i;
            s.found_count = c0 + count[i];
            s.found_before = cb;
            s.found_mass_before = mb;
        }
    }
    __syncthreads();
}

// What a query found: running weight there, and the token (its key, and which of its equals by index, from 1).
struct SampleHit {
    uint64_t mass;
    uint32_t key, rank;
    int index;   // -1: not known, by rank
};

template <int KIND>
__global__ __launch_bounds__(kSampleThreads) void sample_kernel(const SampleArgs p) {
    __shared__ SampleShared s;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int64_t row = blockIdx.x;
    SampleRow<KIND> x = {static_cast<const char*>(p.logits) + row * p.ld * (KIND == 0 ? 4 : 2), p.V};
    if (t < 1 << kExpBits) s.exp2[t] = exp2((double)t / (1 << kExpBits));
    for (int i = t; i < kBuckets; i += kSampleThreads) s.mass[i] = 0, s.count[i] = 0;
    float m = -INFINITY;
    bool bad = false;
    x.each([&](float l, int) { m = fmaxf(m, l), bad = bad || l != l; });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (lane == 0) s.wave32[wave] = __float_as_uint(m);
    const bool none = __syncthreads_or(bad);
    for (int w = 0; w < kSampleWaves; ++w) m = fmaxf(m, __uint_as_float(s.wave32[w]));
    if (none || m == -INFINITY) {   // a NaN, or nothing to take
        if (t == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = NAN;
        }
        return;
    }
    float temperature = p.temperature ? p.temperature[row] : p.temperature1;
    int k = p.top_k ? p.top_k[row] : p.top_k1;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p1, min_p = p.min_p ? p.min_p[row] : p.min_p1;
    if (!(temperature > 0.f)) temperature = 1.f, k = 1;   // the first in order
    SampleScale sc;
    sc.m = m;
    sc.octaves = 128. * M_LOG2E / (double)temperature;
    sc.per_bucket = fminf((float)(sc.octaves * (kBuckets / (128. * kOctaves))), 3e38f);
    const double y_min = min_p > 0.f ? 128. * log2((double)min_p) : -INFINITY;
    __syncthreads();

    // Buckets, and how many tokens min-p leaves.
    uint32_t above = 0;
    x.each([&](float l, int) {
        const int b = sc.bucket(l);
        if (b >= kBuckets) return;
        const double y = sc.exponent(l);
        above += y >= y_min;
        atomicAdd(&s.count[b], 1u);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), (unsigned long long)sc.weight(y, s.exp2));
    });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) above += __shfl_xor(above, d, 64);
    if (lane == 0) s.wave32[wave] = above;
    __syncthreads();
    above = 0;
    for (int w = 0; w < kSampleWaves; ++w) above += s.wave32[w];
    __syncthreads();
    sample_running(s, s.count, s.mass);
    const uint32_t all = s.count[kBuckets - 1];
    const uint64_t all_mass = s.mass[kBuckets - 1];

    int list_lo = 0, list_hi = -1;   // buckets whose tokens are in the list, in order
    auto before_count = [&](int b) { return b ? s.count[b - 1] : 0u; };
    auto before_mass = [&](int b) { return b ? s.mass[b - 1] : 0ull; };

    auto collect = [&](int lo, int hi) {
        for (int i = t; i < kBuckets; i += kSampleThreads) s.cursor[i] = 0;
        __syncthreads();
        const uint32_t start = before_count(lo), n = s.count[hi] - start;
        x.each([&](float l, int i) {
            const int b = sc.bucket(l);
            if (b < lo || b > hi) return;
            s.list.raw[before_count(b) - start + atomicAdd(&s.cursor[b], 1u)] = (uint64_t)~sample_key(l) << 32 | (uint32_t)i;
        });
        __syncthreads();
        for (uint32_t i = t; i < n; i += kSampleThreads) {   // its place among its bucket's
            const uint64_t e = s.list.raw[i];
            const int b = sc.bucket(sample_value(~(uint32_t)(e >> 32)));
            const uint32_t from = before_count(b) - start, to = s.count[b] - start;
            uint32_t place = from;
            for (uint32_t j = from; j < to; ++j) place += s.list.raw[j] < e;
            s.list.sorted[place] = e;
        }
        __syncthreads();
        for (int i = t; i < kSampleList; i += kSampleThreads)
            s.list.run[i] = (uint32_t)i < n ? sc.weight(sc.exponent(sample_value(~(uint32_t)(s.list.sorted[i] >> 32))), s.exp2) : 0ull;
        __syncthreads();
        sample_running(s, nullptr, s.list.run);
        list_lo = lo;
        list_hi = hi;
    };

    auto ask = [&](const SampleQuery& q, bool last) -> SampleHit {
        sample_find(s, s.count, s.mass, 0u, 0ull, q);
        const int b = (int)s.found;
        uint32_t c0 = s.found_before, n = s.found_count - c0;
        uint64_t m0 = s.found_mass_before;
        __syncthreads();
        if (b < list_lo || b > list_hi) {
            if (!last && s.count[b] <= kSampleList) collect(0, b);
            else if (n <= kSampleList) collect(b, b);
        }
        if (b >= list_lo && b <= list_hi) {
            const uint32_t start = before_count(list_lo), len = s.count[list_hi] - start;
            const uint64_t mass0 = before_mass(list_lo);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t i = 2 * t + j;
                if (i < len && q.at(start + i + 1, mass0 + s.list.run[i]) &&
                    (i == 0 || !q.at(start + i, mass0 + s.list.run[i - 1]))) {
                    s.found_entry = s.list.sorted[i];
                    s.found_mass = mass0 + s.list.run[i];
                }
            }
            __syncthreads();
            const SampleHit hit = {s.found_mass, ~(uint32_t)(s.found_entry >> 32), 0, (int)(uint32_t)s.found_entry};
            __syncthreads();
            return hit;
        }
        // More tokens than the list takes: parts of the bucket's keys, from the largest down.
        list_hi = -1, list_lo = 0;
        uint32_t lo = 0, hi = 0xffffffffu;
        while (true) {
            if (t == 0) s.lo = 0xffffffffu, s.hi = 0;
            __syncthreads();
            uint32_t lo1 = 0xffffffffu, hi1 = 0;
            x.each([&](float l, int) {
                const uint32_t key = sample_key(l);
                if (key >= lo && key <= hi && sc.bucket(l) == b) lo1 = min(lo1, key), hi1 = max(hi1, key);
            });
            if (lo1 <= hi1) atomicMin(&s.lo, lo1), atomicMax(&s.hi, hi1);
            __syncthreads();
            lo = s.lo, hi = s.hi;
            if (lo == hi) break;
            int shift = 0;
            while ((hi - lo) >> shift >= (uint32_t)kBuckets) ++shift;
            for (int i = t; i < kBuckets; i += kSampleThreads) s.part.mass[i] = 0, s.part.count[i] = 0;
            __syncthreads();
            x.each([&](float l, int) {
                const uint32_t key = sample_key(l);
                if (key < lo || key > hi || sc.bucket(l) != b) return;
                const uint32_t i = (hi - key) >> shift;
                atomicAdd(&s.part.count[i], 1u);
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.part.mass[i]), (unsigned long long)sc.weight(sc.exponent(l), s.exp2));
            });
            __syncthreads();
            sample_running(s, s.part.count, s.part.mass);
            sample_find(s, s.part.count, s.part.mass, c0, m0, q);
            const uint32_t i = s.found, width = (1u << shift) - 1u;
            n = s.found_count - s.found_before;
            c0 = s.found_before;
            m0 = s.found_mass_before;
            __syncthreads();
            hi -= i << shift;
            lo = hi - lo > width ? hi - width : lo;
        }
        const uint64_t w = sc.weight(sc.exponent(sample_value(lo)), s.exp2);
        uint32_t below = 0, r = n;   // n equals: the first that answers, in (below, r]
        while (r - below > 1) {
            const uint32_t mid = below + (r - below) / 2;
            if (q.at(c0 + mid, m0 + mid * w)) r = mid;
            else below = mid;
        }
        return SampleHit{m0 + r * w, lo, r, -1};
    };

    // What top-k keeps, of that what top-p and min-p keep.
    const uint32_t first_k = k <= 0 ? all : min((uint32_t)k, all);
    const bool with_p = top_p < 1.f;
    const SampleQuery any = {0xffffffffu, INFINITY, false};
    uint64_t kept = all_mass;
    if (with_p && first_k < all) kept = ask(SampleQuery{first_k, any.mass, false}, false).mass;
    const uint32_t most = max(1u, min(first_k, above));
    if (with_p || most < all) kept = ask(SampleQuery{most, with_p ? (double)top_p * (double)kept : any.mass, false}, false).mass;
    const double total = (double)kept;
    const double u = fmax((double)p.u[row], 0.);
    const SampleHit hit = ask(SampleQuery{any.count, fmin(u * total, total * (1. - 0x1p-53)), true}, true);
    int index = hit.index;
    if (index < 0) {   // the hit.rank-th of its equals: ranges of 512 indexes, then the one that holds it
        for (int i = t; i < kBuckets; i += kSampleThreads) s.cursor[i] = 0;
        __syncthreads();
        x.each([&](float l, int i) {
            if (sample_key(l) == hit.key) atomicAdd(&s.cursor[i >> 9], 1u);
        });
        __syncthreads();
        sample_running(s, s.cursor, nullptr);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = 2 * t + j;
            const uint32_t b = i ? s.cursor[i - 1] : 0u;
            if (s.cursor[i] >= hit.rank && b < hit.rank) s.found = i, s.found_before = b;
        }
        __syncthreads();
        const int i = 512 * (int)s.found + t;
        const bool is = t < 512 && i < p.V && sample_key(x.one(i)) == hit.key;
        const uint64_t set = __ballot(is);
        if (lane == 0) s.wave32[wave] = __popcll(set);
        __syncthreads();
        uint32_t place = s.found_before + __popcll(set & ((1ull << lane) - 1ull)) + 1;
        for (int w = 0; w < wave; ++w) place += s.wave32[w];
        if (is && place == hit.rank) s.token = i;
        __syncthreads();
        index = s.token;
    }
    if (t == 0) {
        p.token[row] = index;
        const float l = sample_value(hit.key);
        if (p.logprob)
            p.logprob[row] = (float)((l == m ? 0. : ((double)l - (double)m) / (double)temperature) - log(total * (1. / kUnit)));
    }
}

}  // namespace sfk

extern "C" int sf_sample(const sf_sample_desc* d, void* stream) {
    if (!d || d->rows < 0 || d->V <= 0) return SF_EINVAL;
    if (d->dtype != SF_F32 && d->dtype != SF_BF16 && d->dtype != SF_F16) return SF_ENOTSUP;
    if (d->V > SF_SAMPLE_MAX_VOCAB || d->rows >= 1 << 22) return SF_ENOTSUP;   // a launch counts its threads in 32 bits
    if (d->rows == 0) return SF_OK;
    if (!d->logits || !d->u || !d->token || d->ld < d->V) return SF_EINVAL;
    if (reinterpret_cast<uintptr_t>(d->logits) & (d->dtype == SF_F32 ? 3 : 1)) return SF_EINVAL;
    for (const void* q : {(const void*)d->u, (const void*)d->temperature, (const void*)d->top_k, (const void*)d->top_p,
                          (const void*)d->min_p, (const void*)d->token, (const void*)d->logprob})
        if (reinterpret_cast<uintptr_t>(q) & 3) return SF_EINVAL;
    const sfk::SampleArgs p = {d->logits, d->ld, d->u, d->temperature, d->top_p, d->min_p, d->top_k,
                               d->temperature_all, d->top_p_all, d->min_p_all, d->top_k_all, d->V, d->token, d->logprob};
    const dim3 grid((unsigned)d->rows), block(sfk::kSampleThreads);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (d->dtype == SF_F32) hipLaunchKernelGGL(sfk::sample_kernel<0>, grid, block, 0, s, p);
    else if (d->dtype == SF_BF16) hipLaunchKernelGGL(sfk::sample_kernel<1>, grid, block, 0, s, p);
    else hipLaunchKernelGGL(sfk::sample_kernel<2>, grid, block, 0, s, p);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
