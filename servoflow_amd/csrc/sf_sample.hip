// One token from each row of logits: temperature, top-k, top-p, min-p (gfx950).
//
// With the row's largest logit m a token's weight is 2^43 exp((l - m) / temperature)
// rounded to a whole number, from a table of 2^(j / 128) and four terms of the series
// in 64 bits (1.3e-15 relative).  Sums of weights are sums of whole numbers below
// 2^63 for up to 2^20 tokens: their order does not matter, so a row's token depends
// on the row alone, and neighbours in the running sum differ by far more than it is
// off -- a vocabulary of 131072 in 32 bits would draw another token than 64 bits do
// once in some ten rows.  What is below 2^-44 of the largest counts as nothing (but in
// a logprob near 0, which is nothing but what the others weigh: fine_tail).
//
// Every filter keeps a prefix of the tokens in falling order, so all that is ever
// asked of that order is the first position whose running count or running weight
// passes a number.  Nothing is sorted for it.
//
// 16-bit logits have few values: a row is counted by value, 65536 counts of 16 bits in
// LDS, in one pass that needs no maximum; the values that occur are put together in
// order, each gets its weight once, and the position is a value and a number among its
// equals, whose index one more pass over the row finds in registers.
//
// 32-bit logits, and rows in which that fails (two values, say, that occur more than
// 65535 times), are spread over 2048 buckets of (l - m) / temperature, 1 / 44.5
// octave each, with count and weight of each; the bucket that
// holds the position is found from their running sums, and only its tokens (with
// those above it where they are few) are put in order, in LDS.  A bucket of more than
// 2048 tokens is cut by keys, 2048 parts at a time, until one value is left, of which
// the tokens go by index.
//
// A workgroup takes a row alone in both.  Few long rows of 32 bits are cut into parts
// first: their largest logits, then their buckets added up in memory, two launches
// that the whole card shares, before the one that chooses.
//
// What bounds them (us): 256 rows of 131072 bf16 logits take 40, 18 of them until the
// row is counted (the rows come at 3.7 TB/s, and the counts, one LDS addition for every
// logit, go 8.8 clocks for 64), then a chain of a row's own: the values put in order 4,
// their weights 2, each question 1, the pass for the index 2.  A CU reads 45 GB/s: 50001
// fp32 logits take 6.6 a pass.  Straight code costs, run once by every row: a row of
// 1000 logits took 33 with all loops unrolled, and 14 now.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "sf_device.h"
#include "sf_hip.h"

namespace sfk {

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
constexpr int kBuckets = 2 * kSampleThreads;        // two to a thread
constexpr int kSampleList = 2 * kSampleThreads;     // tokens put in order at a time, two to a thread
constexpr uint32_t kListFromTop = 512;              // so many at most of all buckets above one, too
constexpr int kExpBits = 7;
constexpr float kOctaves = 46.f;                    // 2^-46 and below: no weight
constexpr double kUnit = 8796093022208.;            // 2^43
constexpr double kFaint = -128. * 80.;              // exponents of what is nothing in any sum
// Units of what all others of a row weigh.  They are asked for where they are less than V 2^-24 of the largest (fine_tail),
// within V 2^-44: below 2^64 in units of 2^-70 up to 2^17 tokens, and in units of 2^-67 up to the most there are.
constexpr int kFineTokens = 1 << 17;
constexpr double kFineFew = 0x1p70, kFineMany = 0x1p67;
constexpr double kFineMost = 0x1p-24 + 0x1p-44;   // of each
static_assert(kFineFew * kFineTokens * kFineMost < 0x1p64 && kFineMany * SF_SAMPLE_MAX_VOCAB * kFineMost < 0x1p64, "64 bits");

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
    char* parts;   // of a row cut into parts: SampleParts
    int n_parts;
};

constexpr int kMaxParts = 64;
struct SampleParts {
    uint64_t mass[kBuckets];
    uint32_t count[kBuckets];
    uint64_t above, others;   // as sample_fill's
    float largest[kMaxParts];   // a NaN where there is one
};

struct SampleSums {
    uint64_t mass[kBuckets];     // running, once summed
    uint32_t count[kBuckets];
    uint64_t wave64[kSampleWaves];
    uint32_t wave32[kSampleWaves];
};

struct SampleShared : SampleSums {
    uint32_t cursor[kBuckets];   // a part's tokens; counts of index ranges
    struct {
        uint64_t mass[kBuckets];
        uint32_t count[kBuckets];
    } part;                      // the list by parts of its buckets, or a bucket by keys
    struct {
        uint64_t token[kSampleList];   // ~key << 32 | index: falling order of keys, rising of indexes
        uint64_t weight[kSampleList];
        uint32_t part[kSampleList];
    } list;
    // what one thread found
    uint32_t found, found_count, found_before;
    uint64_t found_mass, found_mass_before, found_entry;
    uint32_t lo, hi;
    int token;
};

// 2^43 2^(j / 128).
__device__ __forceinline__ void sample_table(double* table) {
    if (threadIdx.x < 1 << kExpBits) table[threadIdx.x] = kUnit * exp2((double)threadIdx.x / (1 << kExpBits));
}

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
    // f(logit, index) for every element, each thread its own: one by one, for what is rare.
    template <class F>
    __device__ __forceinline__ void each_slowly(F f) const {
#pragma unroll 1
        for (int i = threadIdx.x; i < V; i += kSampleThreads) f(one(i), i);
    }
    // The same in whole pieces of 16 bytes, AT_ONCE of them under way beside as many that are looked at, and singly what lies
    // before the first and behind the last.  (Many at once keep a row's loads from waiting for each other; what does much
    // with each logit takes few, or no cache of instructions holds it.)
    template <int AT_ONCE, class F>
    __device__ __forceinline__ void each(F f) const {
        pieces_of<AT_ONCE>([&](const u32x4* v, int c0, int head, int pieces) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                const int c = c0 + j * kSampleThreads;
                if (c >= pieces) break;
#pragma unroll
                for (int e = 0; e < E; ++e) f(element(v[j], e), head + c * E + e);
            }
        }, f);
    }

private:
    static __device__ __forceinline__ float element(const u32x4& v, int e) {
        if (KIND == 0) return __uint_as_float(v[e & 3]);
        if (KIND == 1) return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
        return (float)__builtin_bit_cast(_Float16, (uint16_t)(v[e >> 1] >> (16 * (e & 1))));
    }
    template <int AT_ONCE, class Pieces, class F>
    __device__ __forceinline__ void pieces_of(Pieces take, F f) const {
        const int t = threadIdx.x;
        const int size = KIND == 0 ? 4 : 2;
        const int head = min(V, (int)((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / size);
        const int pieces = (V - head) / E, tail = head + pieces * E;
        const u32x4* from = reinterpret_cast<const u32x4*>(base + head * size);
        u32x4 next[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j)
            if (t + j * kSampleThreads < pieces) next[j] = from[t + j * kSampleThreads];
#pragma unroll 1
        for (int c0 = t; c0 < pieces; c0 += AT_ONCE * kSampleThreads) {
            u32x4 v[AT_ONCE];
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                v[j] = next[j];
                const int c = c0 + (AT_ONCE + j) * kSampleThreads;
                if (c < pieces) next[j] = from[c];
            }
            take(v, c0, head, pieces);
        }
        if (t < head) f(one(t), t);
        if (t < V - tail) f(one(tail + t), tail + t);
    }
};

// What a logit counts for.
struct SampleScale {
    float m, per_bucket;           // buckets for twice a difference
    double octaves;                // 128 log2 e / temperature
    // Half of how far it lies above the largest: the whole may be beyond fp32.
    __device__ __forceinline__ float below(float l) const { return l == m ? 0.f : __builtin_fmaf(0.5f, l, -0.5f * m); }
    __device__ __forceinline__ int bucket(float l) const {   // kBuckets and more: no weight
        const float b = -below(l) * per_bucket;
        return b < (float)kBuckets ? (int)b : kBuckets;
    }
    // Bounds of the logits of buckets lo .. hi, 2^-18 of them and of m wider than the roundings of `bucket` ask for.
    __device__ __forceinline__ void range(int lo, int hi, float& from, float& to) const {
        const double step = 2. / (double)per_bucket, slack = fabs((double)m) * 0x1p-18;
        from = per_bucket > 0.f ? (float)((double)m - (double)(hi + 1) * step * (1. + 0x1p-18) - slack) : -INFINITY;
        to = per_bucket > 0.f && lo > 0 ? (float)((double)m - (double)lo * step * (1. - 0x1p-18) + slack) : INFINITY;
        if (fabsf(m) == INFINITY) from = m;
    }
    __device__ __forceinline__ double exponent(float l) const {   // of two, times 128
        return l == m ? 0. : ((double)l - (double)m) * octaves;
    }
    static __device__ __forceinline__ bool in_play(double y) { return y >= -128. * kOctaves; }
    // 0 below the buckets' range.  (A bucket may hold such logits: per_bucket ends at 3e38, so those closer than 1.4e-35 to the
    // largest are in one however small the temperature, and `power` has no value for their exponents.)
    static __device__ __forceinline__ uint64_t weight(double y, const double* table) {
        return rounded(power(fmax(y, -128. * (kOctaves + 1.)), table));
    }
    static __device__ __forceinline__ uint64_t rounded(double w) {
        return (uint64_t)__double_as_longlong(w + 4503599627370496.) & 0xfffffffffffffull;   // + 2^52
    }
    // A weight of a tail, in units of 1 / fine.
    __device__ __forceinline__ uint64_t fine_weight(double y, const double* table, double fine) const {
        return y >= kFaint ? (uint64_t)(power(y, table) * (fine * (1. / kUnit))) : 0ull;
    }
    static __device__ __forceinline__ double power(double y, const double* table) {   // 2^43 2^(y / 128), y from kFaint on
        constexpr double c = M_LN2 / 128., magic = 6755399441055744.;   // 1.5 2^52: the nearest whole number in the low bits
        const double z = y + magic, r = y - (z - magic);
        const uint32_t n = (uint32_t)__double_as_longlong(z);
        const double e = 1. + r * (c + r * (c * c / 2. + r * (c * c * c / 6. + r * (c * c * c * c / 24.))));
        const uint64_t w = (uint64_t)__double_as_longlong(e * table[n & 127u]);   // to be times 2^(n / 128), rounded down
        return __longlong_as_double((long long)((uint64_t)((uint32_t)(w >> 32) + ((n & ~127u) << 13)) << 32 | (uint32_t)w));
    }
};

// Running sums over a wave's lanes (16 lanes: over each row), vector instructions alone.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_or_0(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp_or_0(uint64_t x) {
    return (uint64_t)dpp_or_0<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 | dpp_or_0<CTRL, ROWS>((uint32_t)x);
}
template <class T>
__device__ __forceinline__ T running16(T x) {
    x += dpp_or_0<0x111, 0xf>(x);   // row_shr 1, 2, 4, 8
    x += dpp_or_0<0x112, 0xf>(x);
    x += dpp_or_0<0x114, 0xf>(x);
    x += dpp_or_0<0x118, 0xf>(x);
    return x;
}
template <class T>
__device__ __forceinline__ T running64(T x) {
    x = running16(x);
    x += dpp_or_0<0x142, 0xa>(x);   // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
    x += dpp_or_0<0x143, 0xc>(x);
    return x;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
__device__ __forceinline__ uint64_t lane_of(uint64_t x, int lane) {
    return (uint64_t)lane_of((uint32_t)(x >> 32), lane) << 32 | lane_of((uint32_t)x, lane);
}
// What the waves before `wave` put into sums, and all of them.
template <class T>
__device__ __forceinline__ T before_wave(const T* sums, int wave, T& all) {
    const T own = sums[threadIdx.x & (kSampleWaves - 1)], run = running16(own);
    all = lane_of(run, kSampleWaves - 1);
    return lane_of(run, wave) - lane_of(own, wave);
}

// A barrier for what is in LDS: loads from memory stay under way.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Running sums over 2048 counts and weights (either may be null), two to a thread.
__device__ __forceinline__ void sample_running(SampleSums& s, uint32_t* count, uint64_t* mass) {
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    uint32_t c0 = 0, c = 0, all_c;
    uint64_t m0 = 0, m = 0, all_m;
    if (count) c0 = count[2 * t], c = c0 + count[2 * t + 1];
    if (mass) m0 = mass[2 * t], m = m0 + mass[2 * t + 1];
    uint32_t ci = running64(c);
    uint64_t mi = running64(m);
    if (lane == 63) s.wave32[wave] = ci, s.wave64[wave] = mi;
    __syncthreads();
    ci += before_wave(s.wave32, wave, all_c);
    mi += before_wave(s.wave64, wave, all_m);
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
    int index;   // -1: not known, by rank (else the rank says nothing)
};

// The first of n equal tokens of weight w, behind (c0, m0), that answers q; the last one does.
__device__ __forceinline__ uint32_t sample_among_equals(const SampleQuery& q, uint32_t n, uint32_t c0, uint64_t m0, uint64_t w) {
    uint32_t below = 0, r = n;
    while (r - below > 1) {
        const uint32_t mid = below + (r - below) / 2;
        if (q.at(c0 + mid, m0 + mid * w)) r = mid;
        else below = mid;
    }
    return r;
}

// The parameters of a row.
struct SampleRule {
    float temperature, top_p;
    int k;
    SampleScale sc;
    double y_min;   // min-p: exponents from here on
    double fine_all;
    __device__ __forceinline__ void read(const SampleArgs& p, int64_t row) {
        temperature = p.temperature ? p.temperature[row] : p.temperature1;
        k = p.top_k ? p.top_k[row] : p.top_k1;
        top_p = p.top_p ? p.top_p[row] : p.top_p1;
        const float min_p = p.min_p ? p.min_p[row] : p.min_p1;
        if (!(temperature > 0.f)) temperature = 1.f, k = 1;   // the first in order
        y_min = min_p > 0.f ? 128. * (log2((double)min_p) - M_LOG2E * 0x1p-54) : -INFINITY;   // what 64 bits round to min_p reaches it
        fine_all = p.V <= kFineTokens ? kFineFew : kFineMany;
        sc.octaves = 128. * M_LOG2E / (double)temperature;
        sc.per_bucket = (float)fmin(sc.octaves * (kBuckets / (64. * kOctaves)), 3e38);
    }
    // The three questions that a row's token takes: what top-k keeps, what top-p keeps of that, and where u falls.  What
    // min-p leaves is a beginning of the order too: `above`, its weight.  ask(query, last) answers.
    template <class Ask>
    __device__ __forceinline__ SampleHit token(uint32_t all, uint64_t all_mass, uint64_t above, float u, uint64_t& kept, SampleHit& end,
                                               Ask ask) const {
        const uint32_t first_k = k <= 0 ? all : min((uint32_t)k, all);
        const bool with_p = top_p < 1.f;
        SampleHit hit = {};
        kept = all_mass;
        end.rank = 0;
#pragma unroll 1
        for (int step = 0; step < 3; ++step) {
            SampleQuery q = {0xffffffffu, INFINITY, false};
            if (step == 0) {
                if (!with_p || first_k >= all) continue;
                q.count = first_k;
            } else if (step == 1) {
                if (!with_p && first_k >= all && k != 1) continue;   // (the first alone has it all, whatever lies below the buckets)
                q.count = first_k;
                if (with_p) q.mass = (double)top_p * (double)kept;
            } else {
                kept = min(kept, max(above, (uint64_t)kUnit));   // one at least
                const double total = (double)kept;
                q.mass = fmin(fmax((double)u, 0.) * total, total * (1. - 0x1p-53));
                q.strict = true;
            }
            hit = ask(q, step == 2);
            if (step < 2) kept = hit.mass, end = hit;
        }
        return hit;
    }
    // A largest token's share of nearly all needs what the others weigh to more digits than the questions do: V weights held
    // to 2^-44 are off by up to V 2^-44 in all, and a logprob of -1e-6 is to be as exact as others.  So where V others at most
    // weigh less than V 2^-24 they are summed once more, in units of 2^-75, or 2^-67 from 2^-12 on.  `end` is the last token that
    // top-k and top-p keep (rank 0: all are kept), `top` the largest.  0: the logprob of `kept` will do.
    __device__ __forceinline__ double fine_tail(const SampleHit& hit, const SampleHit& end, uint32_t top, uint64_t kept, int V) const {
        const uint64_t others = kept - (uint64_t)kUnit;
        if (hit.key != top || (end.rank && end.key == top) || others >= (uint64_t)V << 19) return 0.;
        return others < 1ull << 31 ? 0x1p75 : 0x1p67;
    }
    static __device__ __forceinline__ float tail_logprob(uint64_t tail, double fine) { return (float)-log1p((double)tail / fine); }
    __device__ __forceinline__ float logprob(float l, uint64_t kept) const {
        return (float)((l == sc.m ? 0. : ((double)l - (double)sc.m) / (double)temperature) - log((double)kept * (1. / kUnit)));
    }
};

// The index of the rank-th token of a key: counts of ranges of 512 indexes, then the range that holds it.
template <int KIND>
__device__ __forceinline__ int sample_nth(SampleShared& s, const SampleRow<KIND>& x, uint32_t key, uint32_t rank) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    for (int i = t; i < kBuckets; i += kSampleThreads) s.cursor[i] = 0;
    __syncthreads();
    x.template each<2>([&](float l, int i) {
        if (sample_key(l) == key) atomicAdd(&s.cursor[i >> 9], 1u);
    });
    __syncthreads();
    sample_running(s, s.cursor, nullptr);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int i = 2 * t + j;
        const uint32_t b = i ? s.cursor[i - 1] : 0u;
        if (s.cursor[i] >= rank && b < rank) s.found = i, s.found_before = b;
    }
    __syncthreads();
    const int i = 512 * (int)s.found + t;
    const bool is = t < 512 && i < x.V && sample_key(x.one(i)) == key;
    const uint64_t set = __ballot(is);
    if (lane == 0) s.wave32[wave] = __popcll(set);
    __syncthreads();
    uint32_t place = s.found_before + __popcll(set & ((1ull << lane) - 1ull)) + 1;
    for (int w = 0; w < wave; ++w) place += s.wave32[w];
    if (is && place == rank) s.token = i;
    __syncthreads();
    return s.token;
}

// The largest of a workgroup's logits, a NaN if there is one.
template <int KIND>
__device__ __forceinline__ float sample_largest(SampleSums& s, const SampleRow<KIND>& x) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    float m = -INFINITY;
    bool bad = false;
    x.template each<4>([&](float l, int) { m = fmaxf(m, l), bad = bad || l != l; });
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    if (lane == 0) s.wave32[wave] = __float_as_uint(m);
    const bool none = __syncthreads_or(bad);
    m = __uint_as_float(s.wave32[lane & (kSampleWaves - 1)]);
#pragma unroll
    for (int d = kSampleWaves / 2; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    return none ? NAN : m;
}

// Adds a workgroup's logits to the buckets; the weight that min-p leaves of them.  Counts are for top-k alone, and for
// lists of few tokens; without them a bucket's weight tells how many it holds at most.  others: what all but the largest
// weigh, of those that min-p leaves, in units of 1 / rule.fine_all, each thread's to the nearest (of a row in parts V / 4 threads at
// most: V 2^-70); more than 64 bits hold where it is not used.
template <int KIND>
__device__ __forceinline__ uint64_t sample_fill(SampleSums& s, const double* table, const SampleRow<KIND>& x, const SampleRule& rule,
                                                uint64_t& others) {
    const SampleScale& sc = rule.sc;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const bool counted = rule.k > 0, with_min_p = rule.y_min > -INFINITY;
    uint64_t above = 0;
    double rest = 0.;
    for (int i = t; i < kBuckets; i += kSampleThreads) s.mass[i] = 0, s.count[i] = 0;
    __syncthreads();
    x.template each<2>([&](float l, int) {
        const int b = sc.bucket(l);
        const double y = sc.exponent(l);
        if (!(y >= kFaint)) return;
        const double exact = sc.power(y, table);
        if (y >= rule.y_min && l != sc.m) rest += exact;
        if (b >= kBuckets) return;
        const uint64_t w = sc.rounded(exact);
        atomicAdd(reinterpret_cast<unsigned long long*>(&s.mass[b]), (unsigned long long)w);
        if (counted) atomicAdd(&s.count[b], 1u);
        if (with_min_p) above += y >= rule.y_min ? w : 0ull;
    });
    if (with_min_p) {
        above = running64(above);
        if (lane == 63) s.wave64[wave] = above;
        __syncthreads();
        before_wave(s.wave64, wave, above);
    }
    __syncthreads();
    others = running64((uint64_t)(fmin(rest * (rule.fine_all / kUnit), 0x1p63) + 0.5));
    if (lane == 63) s.wave64[wave] = others;
    __syncthreads();
    before_wave(s.wave64, wave, others);
    __syncthreads();
    return above;
}

// A row's token from its buckets (rule.sc.m set; above: as sample_fill's).
template <int KIND>
__device__ __forceinline__ void sample_by_buckets(const SampleArgs& p, SampleShared& s, const double* table, const SampleRow<KIND>& x,
                                                  const SampleRule& rule, uint64_t above, uint64_t others, int64_t row) {
    const int t = threadIdx.x;
    const SampleScale& sc = rule.sc;
    const bool counted = rule.k > 0;
    if (!(rule.y_min > -INFINITY)) above = ~0ull;
    sample_running(s, s.count, s.mass);

    int list_lo = 0, list_hi = -1;   // buckets whose tokens are in the list, in order
    auto before_count = [&](int b) { return b ? s.count[b - 1] : 0u; };   // 0 where nothing is counted
    auto before_mass = [&](int b) { return b ? s.mass[b - 1] : 0ull; };

    // Tokens of the buckets lo .. hi, and their sums by 2048 parts of these; how many there are (more than kSampleList: no
    // list).
    auto collect = [&](int lo, int hi) {
        for (int i = t; i < kBuckets; i += kSampleThreads) s.part.mass[i] = 0, s.part.count[i] = 0;
        if (t == 0) s.lo = 0;
        float from, to;   // the buckets' logits lie between them
        sc.range(lo, hi, from, to);
        const float finer = (float)kBuckets / (float)(hi - lo + 1);
        __syncthreads();
        x.template each<2>([&](float l, int i) {
            if (!(l >= from && l <= to)) return;
            const uint32_t at = atomicAdd(&s.lo, 1u);
            if (at < kSampleList) s.list.token[at] = (uint64_t)~sample_key(l) << 32 | (uint32_t)i;
        });
        __syncthreads();
        const uint32_t n = s.lo;   // a few of the buckets beside them among them: they belong to no part
        if (n > kSampleList) {
            __syncthreads();   // s.lo is read: the parts of its keys begin with it
            return n;
        }
        for (uint32_t i = t; i < n; i += kSampleThreads) {
            const float l = sample_value(~(uint32_t)(s.list.token[i] >> 32));
            const int b = sc.bucket(l);
            const uint64_t w = b >= lo && b <= hi ? sc.weight(sc.exponent(l), table) : 0ull;
            const uint32_t part = b >= lo && b <= hi ? min((int)((-sc.below(l) * sc.per_bucket - (float)lo) * finer), kBuckets - 1) : kBuckets;
            s.list.weight[i] = w;
            s.list.part[i] = part;
            if (part == kBuckets) continue;
            atomicAdd(&s.part.count[part], 1u);
            atomicAdd(reinterpret_cast<unsigned long long*>(&s.part.mass[part]), (unsigned long long)w);
        }
        __syncthreads();
        sample_running(s, s.part.count, s.part.mass);
        list_lo = lo;
        list_hi = hi;
        return n;
    };

    uint32_t len = 0;   // of the list
    auto ask = [&](const SampleQuery& q, bool last) -> SampleHit {
        sample_find(s, s.count, s.mass, 0u, 0ull, q);
        const int b = (int)s.found;
        uint32_t c0 = s.found_before, n = 0;
        uint64_t m0 = s.found_mass_before;
        if (!counted) {   // at most (`collect` counts them where buckets are wider than `least` takes them for, as `weight` says)
            const double least = (double)sc.weight(-128. * (double)(b + 1) * (kOctaves / kBuckets), table) * (1. - 0x1p-14) - 1.;
            const double most = least > 0. ? (double)(s.mass[b] - m0) / least : 1e9;
            n = most < 1e9 ? (uint32_t)most : 1000000000u;
        } else {
            n = s.found_count - c0;
        }
        __syncthreads();
        if (b < list_lo || b > list_hi) {
            list_hi = -1, list_lo = 0;
            if (n <= kSampleList) len = collect(!last && counted && s.count[b] <= kListFromTop ? 0 : b, b);
        }
        if (b >= list_lo && b <= list_hi) {
            if (t == 0) s.hi = 0;
            sample_find(s, s.part.count, s.part.mass, before_count(list_lo), before_mass(list_lo), q);
            const uint32_t part = s.found, start = s.found_before;
            const uint64_t mass0 = s.found_mass_before;
            for (uint32_t i = t; i < len; i += kSampleThreads)
                if (s.list.part[i] == part) s.cursor[atomicAdd(&s.hi, 1u)] = i;
            __syncthreads();
            const uint32_t few = s.hi;   // in order: each looks at every other
            for (uint32_t i = t; i < few; i += kSampleThreads) {
                const uint64_t e = s.list.token[s.cursor[i]], w = s.list.weight[s.cursor[i]];
                uint32_t c = start;
                uint64_t m = mass0;
                for (uint32_t j = 0; j < few; ++j)
                    if (s.list.token[s.cursor[j]] < e) ++c, m += s.list.weight[s.cursor[j]];
                if (q.at(c + 1, m + w) && (c == start || !q.at(c, m))) {
                    s.found_entry = e;
                    s.found_mass = m + w;
                }
            }
            __syncthreads();
            const SampleHit hit = {s.found_mass, ~(uint32_t)(s.found_entry >> 32), 1, (int)(uint32_t)s.found_entry};
            __syncthreads();
            return hit;
        }
        // More tokens than the list takes: parts of the bucket's keys, from the largest down.
        uint32_t lo = 0, hi = 0xffffffffu;
        if (!counted) n = (uint32_t)x.V;   // of a bucket of one value: the weight asked for tells which
        while (true) {
            if (t == 0) s.lo = 0xffffffffu, s.hi = 0;
            __syncthreads();
            uint32_t lo1 = 0xffffffffu, hi1 = 0;
            x.each_slowly([&](float l, int) {
                const uint32_t key = sample_key(l);
                if (key >= lo && key <= hi && sc.bucket(l) == b) lo1 = min(lo1, key), hi1 = max(hi1, key);
            });
            if (lo1 <= hi1) atomicMin(&s.lo, lo1), atomicMax(&s.hi, hi1);
            __syncthreads();
            lo = s.lo, hi = s.hi;
            if (lo >= hi) break;
            int shift = 0;
            while ((hi - lo) >> shift >= (uint32_t)kBuckets) ++shift;
            for (int i = t; i < kBuckets; i += kSampleThreads) s.part.mass[i] = 0, s.part.count[i] = 0;
            __syncthreads();
            x.each_slowly([&](float l, int) {
                const uint32_t key = sample_key(l);
                if (key < lo || key > hi || sc.bucket(l) != b) return;
                const uint32_t i = (hi - key) >> shift;
                atomicAdd(&s.part.count[i], 1u);
                atomicAdd(reinterpret_cast<unsigned long long*>(&s.part.mass[i]), (unsigned long long)sc.weight(sc.exponent(l), table));
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
        const uint64_t w = sc.weight(sc.exponent(sample_value(lo)), table);
        const uint32_t r = sample_among_equals(q, n, c0, m0, w);
        return SampleHit{m0 + r * w, lo, r, -1};
    };

    uint64_t kept;
    SampleHit end;
    const uint32_t all = counted ? s.count[kBuckets - 1] : 0xffffffffu;
    const SampleHit hit = rule.token(all, s.mass[kBuckets - 1], above, p.u[row], kept, end, ask);
    const int index = hit.index >= 0 ? hit.index : sample_nth(s, x, hit.key, hit.rank);
    if (t == 0) p.token[row] = index;
    if (!p.logprob) return;
    // All others were summed with the buckets; those that top-k or top-p keep take one more pass, which is rare (37 rows of
    // 50001 with temperature alone take 2 us more for the sums, and took 15 more for such a pass).
    const double fine = rule.fine_tail(hit, end, sample_key(sc.m), kept, end.rank && counted ? (int)min((int64_t)8 * rule.k, (int64_t)x.V) : x.V);
    if (fine == 0. || end.rank == 0) {
        const float y = fine == 0. || end.rank ? rule.logprob(sample_value(hit.key), kept) : rule.tail_logprob(others, rule.fine_all);
        if (t == 0) p.logprob[row] = y;
        return;
    }
    uint64_t tail = 0;
    x.template each<2>([&](float l, int i) {
        const uint32_t key = sample_key(l);
        if (l == sc.m || (end.rank && (key < end.key || (key == end.key && i > end.index)))) return;   // (index -1: below)
        const double y = sc.exponent(l);
        if (y >= rule.y_min) tail += sc.fine_weight(y, table, fine);
    });
    if (t == 0 && end.rank && end.index < 0) {
        const double y = sc.exponent(sample_value(end.key));
        if (y >= rule.y_min) tail += end.rank * sc.fine_weight(y, table, fine);
    }
    tail = running64(tail);
    __syncthreads();
    if ((t & 63) == 63) s.wave64[t >> 6] = tail;
    __syncthreads();
    before_wave(s.wave64, __builtin_amdgcn_readfirstlane(t >> 6), tail);
    if (t == 0) p.logprob[row] = rule.tail_logprob(tail, fine);
}

// A row that has no token: a NaN, or nothing to take.
__device__ __forceinline__ bool sample_none(const SampleArgs& p, float m, int64_t row) {
    const bool none = !(m > -INFINITY);
    if (none && threadIdx.x == 0) {
        p.token[row] = -1;
        if (p.logprob) p.logprob[row] = NAN;
    }
    return none;
}

template <int KIND>
__device__ __forceinline__ void sample_row(const SampleArgs& p, SampleShared& s, double* table, int64_t row) {
    const SampleRow<KIND> x = {static_cast<const char*>(p.logits) + row * p.ld * (KIND == 0 ? 4 : 2), p.V};
    SampleRule rule;
    rule.read(p, row);
    sample_table(table);
    rule.sc.m = sample_largest(s, x);
    if (sample_none(p, rule.sc.m, row)) return;
    uint64_t others;
    const uint64_t above = sample_fill(s, table, x, rule, others);
    sample_by_buckets(p, s, table, x, rule, above, others, row);
}

__global__ __launch_bounds__(kSampleThreads) void sample_f32_kernel(const SampleArgs p) {
    __shared__ SampleShared s;
    __shared__ double table[1 << kExpBits];
    sample_row<0>(p, s, table, blockIdx.x);
}

// ------------------------------------------------------------------ in parts

// Part `part` of a row: whole 4096 bytes of it, but for the first and the last.
__device__ __forceinline__ SampleRow<0> sample_part(const SampleArgs& p, int64_t row, int part) {
    const int each = ((p.V + p.n_parts - 1) / p.n_parts + 1023) & ~1023, from = min(p.V, part * each);
    return SampleRow<0>{static_cast<const char*>(p.logits) + (row * p.ld + from) * 4, min(each, p.V - from)};
}

// The parts' largest logits; and the row's sums are cleared, each part a share.
__global__ __launch_bounds__(kSampleThreads) void sample_parts_largest_kernel(const SampleArgs p) {
    __shared__ SampleSums s;
    const int64_t row = blockIdx.x / p.n_parts;
    const int part = blockIdx.x % p.n_parts;
    SampleParts* sums = reinterpret_cast<SampleParts*>(p.parts) + row;
    for (int i = part * kSampleThreads + threadIdx.x; i < kBuckets; i += p.n_parts * kSampleThreads) sums->mass[i] = 0, sums->count[i] = 0;
    if (part == 0 && threadIdx.x == 0) sums->above = sums->others = 0;
    const float m = sample_largest(s, sample_part(p, row, part));
    if (threadIdx.x == 0) sums->largest[part] = m;
}

// The row's largest, of its parts'.
__device__ __forceinline__ float sample_parts_largest(const SampleArgs& p, const SampleParts* sums) {
    const int lane = threadIdx.x & 63;
    float m = lane < p.n_parts ? sums->largest[lane] : -INFINITY;
    const bool none = __any(m != m);
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
    return none ? NAN : m;
}

__global__ __launch_bounds__(kSampleThreads) void sample_parts_fill_kernel(const SampleArgs p) {
    __shared__ SampleSums s;
    __shared__ double table[1 << kExpBits];
    const int64_t row = blockIdx.x / p.n_parts;
    SampleParts* sums = reinterpret_cast<SampleParts*>(p.parts) + row;
    SampleRule rule;
    rule.read(p, row);
    rule.sc.m = sample_parts_largest(p, sums);
    if (!(rule.sc.m > -INFINITY)) return;
    sample_table(table);
    uint64_t others;
    const uint64_t above = sample_fill(s, table, sample_part(p, row, blockIdx.x % p.n_parts), rule, others);
    for (int i = threadIdx.x; i < kBuckets; i += kSampleThreads) {
        if (s.mass[i]) atomicAdd(reinterpret_cast<unsigned long long*>(&sums->mass[i]), (unsigned long long)s.mass[i]);
        if (s.count[i]) atomicAdd(&sums->count[i], s.count[i]);
    }
    if (threadIdx.x == 0) {
        if (above) atomicAdd(reinterpret_cast<unsigned long long*>(&sums->above), (unsigned long long)above);
        if (others) atomicAdd(reinterpret_cast<unsigned long long*>(&sums->others), (unsigned long long)others);
    }
}

__global__ __launch_bounds__(kSampleThreads) void sample_parts_choose_kernel(const SampleArgs p) {
    __shared__ SampleShared s;
    __shared__ double table[1 << kExpBits];
    const int64_t row = blockIdx.x;
    const SampleParts* sums = reinterpret_cast<const SampleParts*>(p.parts) + row;
    SampleRule rule;
    rule.read(p, row);
    rule.sc.m = sample_parts_largest(p, sums);
    if (sample_none(p, rule.sc.m, row)) return;
    sample_table(table);
    for (int i = threadIdx.x; i < kBuckets; i += kSampleThreads) s.mass[i] = sums->mass[i], s.count[i] = sums->count[i];
    __syncthreads();
    sample_by_buckets(p, s, table, SampleRow<0>{static_cast<const char*>(p.logits) + row * p.ld * 4, p.V}, rule, sums->above, sums->others, row);
}

// In how many parts.  Two more launches have to pay for themselves, the sooner the fewer rows share the card; a part
// has 4096 logits at least, and the parts of all rows make up two workgroups a CU.  us by one workgroup a row and in parts
// (temperature alone): 1 x 16384 17.0, 19.9; 1 x 32768 23.0, 21.1; 1 x 131072 58.0, 26.5; 16 x 32768 24.1, 22.7; 37 x 50001
// 30.9, 28.2; 64 x 32768 25.4, 27.9; 100 x 131072 67.9, 52.9; 160 x 131072 70.1, 65.5; 250 x 131072 86.4, 93.3.
static inline int sample_parts(int rows, int V, int dtype) {
    if (dtype != SF_F32 || V < 28672 + 512 * (int64_t)rows) return 1;
    return std::max(1, std::min({V / 4096, 512 / rows, kMaxParts}));
}

// --------------------------------------------------------------- by value

constexpr int kHeld = 16;             // pieces of 16 bytes that a thread keeps: 131072 tokens of a row
constexpr int kOverflow = -2;         // a token that is still to be found
constexpr int kCommonFrom = 1024;     // rows of as many are looked over for a value that many tokens share
constexpr uint32_t kMaxTies = 1024;   // equals that are told apart in a list
constexpr uint32_t kValueList = 6656;   // values beside the counts

struct SampleValues {
    uint32_t bins[1 << 15];        // two counts each: falling keys 2 i and 2 i + 1
    uint32_t beside[kValueList];   // the values that occur, key << 16 | count; more than that take the counts' place, if they fit
    uint64_t wave64[kSampleWaves];
    uint32_t wave32[kSampleWaves], tokens[kSampleWaves], steps[128];
    struct Hit {
        uint64_t mass;
        uint32_t key, rank, equals;
    } hits[3];
    uint64_t above;
    uint32_t ties, nan, fail, shared_by, common;
    int token;
};

typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Falling keys of two 16-bit floats: whole numbers in falling order (-0 behind 0).
__device__ __forceinline__ uint32_t sample_falling(uint32_t w) {
    const uint32_t minus = __builtin_bit_cast(uint32_t, __builtin_bit_cast(s16x2, w) >> 15);
    return w ^ (~minus & 0x7fff7fffu);
}

template <int KIND>   // 1 bf16, 2 fp16
__global__ __launch_bounds__(kSampleThreads) void sample_16_kernel(const SampleArgs p) {
    __shared__ union {
        SampleShared nth;
        SampleValues values;
    } shared;
    __shared__ double table[1 << kExpBits];
    constexpr uint32_t kInf = KIND == 1 ? 0x7fu : 0x3ffu, kNegInf = 0xffffu - kInf;   // falling keys of the infinities
    constexpr uint32_t kMinusZero = 0x8000, kNoKey = 0x10000;
    SampleValues& s = shared.values;
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int64_t row = blockIdx.x;
    const SampleRow<KIND> x = {static_cast<const char*>(p.logits) + row * p.ld * 2, p.V};
    const int head = min(p.V, (int)((16 - (reinterpret_cast<uintptr_t>(x.base) & 15)) & 15) / 2);
    const int pieces = (p.V - head) / 8, tail = head + pieces * 8;
    const u32x4* from = reinterpret_cast<const u32x4*>(x.base + head * 2);
    const uint16_t some = wave == 0 && p.V >= kCommonFrom ? reinterpret_cast<const uint16_t*>(x.base)[(int)((int64_t)lane * p.V >> 6)] : 0;
    u32x4 held[kHeld];
    const bool in_head = t < head, in_tail = t < p.V - tail;
    const uint32_t first = in_head ? reinterpret_cast<const uint16_t*>(x.base)[t] : 0u;
    const uint32_t last = in_tail ? reinterpret_cast<const uint16_t*>(x.base)[tail + t] : 0u;
    SampleRule rule;
    rule.read(p, row);
    // keys: the key in the low half (what is above it does not matter)
    auto count1 = [&](uint32_t keys) __attribute__((always_inline)) {
        atomicAdd(reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(s.bins) + (keys << 1 & 0x1fffcu)), 1u << (keys << 4 & 16u));
    };
    // Counted apart: -infinity (`none`, and the NaN behind it), and one value that many tokens share, as a row's masked ones
    // do (`common`; of 64 tokens from all over the row, one that two neighbours and twelve in all have).  In their
    // places among the others they would be added one by one, and pass 16 bits: 256 rows of 131072 bf16, all but 2% of them
    // -10000, take 48 us, and took 184 so.
    uint32_t common = kNoKey, shared_by = 0, none = 0;
    bool nan = false;
    auto count_any = [&](uint32_t key) __attribute__((always_inline)) {
        if (key < kNegInf && key != common) count1(key);
        shared_by += key == common;
        none += key >= kNegInf;
        nan = nan || key > kNegInf;   // of either sign: the others are below kInf, and counted
    };
    auto count8 = [&](const u32x4& v) __attribute__((always_inline)) {
        uint32_t k[4];
        u16x2 most = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            k[e] = sample_falling(v[e]);
            most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, k[e]));
        }
        if (common != kNoKey || __any(most[0] >= kNegInf || most[1] >= kNegInf)) {
#pragma unroll 1
            for (int e = 0; e < 8; ++e) {
                const uint32_t x01 = e & 2 ? k[1] : k[0], x23 = e & 2 ? k[3] : k[2];
                count_any((e & 4 ? x23 : x01) >> (16 * (e & 1)) & 0xffffu);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                count1(k[e]);
                count1(k[e] >> 16);
            }
        }
    };
    auto clear = [&]() __attribute__((always_inline)) {
        sample_table(table);
#pragma unroll
        for (int i = 0; i < 8; ++i) reinterpret_cast<u32x4*>(s.bins)[t + i * kSampleThreads] = u32x4{0, 0, 0, 0};
        if (wave == 0) {
            if (p.V >= kCommonFrom) {
                const uint32_t key = sample_falling(some) & 0xffffu;
                uint64_t twice = __ballot(key == dpp_or_0<0x111, 0xf>(key));   // as the lane before: hardly any without such a value
                for (; twice && common == kNoKey; twice &= twice - 1) {
                    const uint32_t k = lane_of(key, __builtin_ctzll(twice));
                    if (__popcll(__ballot(key == k)) >= 12 && k < kNegInf && k != kMinusZero) common = k;
                }
            }
            if (lane == 0) s.common = common, s.shared_by = 0;
        }
        lds_barrier();
        common = __builtin_amdgcn_readfirstlane(s.common);
    };
    if (pieces > kHeld / 2 * kSampleThreads) {   // all loads at once, the last piece again behind it: each is waited for by itself
#pragma unroll
        for (int j = 0; j < kHeld; ++j) held[j] = from[min(t + j * kSampleThreads, pieces - 1)];
        clear();
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (t + j * kSampleThreads < pieces) count8(held[j]);
        for (int c = t + kHeld * kSampleThreads; c < pieces; c += kSampleThreads) count8(from[c]);
    } else {
#pragma unroll
        for (int j = 0; j < kHeld / 2; ++j) {
            if (j * kSampleThreads >= pieces) break;   // (at once, not piece by piece)
            if (t + j * kSampleThreads < pieces) held[j] = from[t + j * kSampleThreads];
        }
        clear();
#pragma unroll
        for (int j = 0; j < kHeld / 2; ++j) {
            if (j * kSampleThreads >= pieces) break;
            if (t + j * kSampleThreads < pieces) count8(held[j]);
        }
    }
    if (in_head) count_any(sample_falling(first) & 0xffffu);
    if (in_tail) count_any(sample_falling(last) & 0xffffu);
    if (common != kNoKey) {
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) shared_by += __shfl_xor(shared_by, d, 64);
        if (lane == 0) atomicAdd(&s.shared_by, shared_by);
    }
    __syncthreads();
    bool fail = false;
    if (t == 0) {   // -0, the first of its count, counts as 0, the second of the one before
        const uint32_t minus = s.bins[0x4000] & 0xffffu;
        s.bins[0x4000] &= 0xffff0000u;
        fail = (s.bins[0x3fff] >> 16) + minus > 0xffffu;
        s.bins[0x3fff] += minus << 16;
        s.above = s.ties = s.nan = s.fail = 0;
        if (s.shared_by) {   // and that value's one, for it to be among those that occur
            uint32_t& two = s.bins[common >> 1];
            const int at = 16 * (common & 1);
            s.shared_by += two >> at & 0xffffu;
            two = (two & ~(0xffffu << at)) | 1u << at;
        }
    }
    __syncthreads();
    const uint32_t many = s.shared_by;
    auto tokens_of = [&](uint32_t e) __attribute__((always_inline)) { return e >> 16 == common ? many : e & 0xffffu; };

    // The values that occur, in order: 128 times 256 counts of two values, which the waves deal.  (Most hold nothing: a
    // row's values are a few thousand, side by side.)
    uint32_t tokens = none;
    if (t == 0 && many) tokens += many - 1;
    auto occur = [](const u32x4& v) __attribute__((always_inline)) {
        uint32_t k = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) k += ((v[e] & 0xffffu) ? 1u : 0u) + (v[e] >> 16 ? 1u : 0u);
        return k;
    };
    const u32x4* counts = reinterpret_cast<const u32x4*>(s.bins) + 64 * wave + lane;
    auto key_of = [&](int i) __attribute__((always_inline)) { return 8u * (64 * (16 * i + wave) + lane); };
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
        u32x4 v = counts[1024 * i];
        uint32_t mine = 0;
        if (__any((v[0] | v[1] | v[2] | v[3]) != 0)) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                tokens += (v[e] & 0xffffu) + (v[e] >> 16);
                nan = nan || ((v[e] & 0xffffu) && key_of(i) + 2 * e < kInf) || (v[e] >> 16 && key_of(i) + 2 * e + 1 < kInf);
            }
            mine = lane_of(running64(occur(v)), 63);
        }
        if (lane == 0) s.steps[16 * i + wave] = mine;
    }
    tokens = running64(tokens);
    if (lane == 63) s.tokens[wave] = tokens;
    if (nan) s.nan = 1;
    if (fail) s.fail = 1;
    __syncthreads();
    before_wave(s.tokens, wave, tokens);
    const uint32_t own0 = s.steps[lane], own1 = s.steps[64 + lane];
    const uint32_t to0 = running64(own0), to1 = running64(own1) + lane_of(to0, 63), n = lane_of(to1, 63);
    if (s.fail || tokens != (uint32_t)p.V) {   // a count that passed 16 bits: the sum of all is too small
        if (t == 0) p.token[row] = kOverflow;
        return;
    }
    if (s.nan || n == 0) {
        if (t == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = NAN;
        }
        return;
    }
    uint32_t* list = s.beside;
    auto put = [&](const u32x4& v, int i) __attribute__((always_inline)) {
        const uint32_t k = occur(v), run = running64(k), key = key_of(i);
        const int step = 16 * i + wave;
        uint32_t place = (step < 64 ? lane_of(to0 - own0, step) : lane_of(to1 - own1, step - 64)) + run - k;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (v[e] & 0xffffu) list[place++] = (key + 2 * e) << 16 | (v[e] & 0xffffu);
            if (v[e] >> 16) list[place++] = (key + 2 * e + 1) << 16 | v[e] >> 16;
        }
    };
    const bool listed = n <= sizeof(s.bins) / sizeof(s.bins[0]);
    if (n <= kValueList) {
#pragma unroll 1
        for (int i = 0; i < 8; ++i) {
            const u32x4 v = counts[1024 * i];
            if (__any((v[0] | v[1] | v[2] | v[3]) != 0)) put(v, i);
        }
    } else if (listed) {   // in the counts' place, once they are in registers
        list = s.bins;
        u32x4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = counts[1024 * i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) put(v[i], i);
    }
    __syncthreads();
    // Value i of them, or of all keys.
    const uint32_t values = listed ? n : 65536u;
    auto entry = [&](uint32_t i) __attribute__((always_inline)) {
        return listed ? list[i] : i << 16 | (s.bins[i >> 1] >> (16 * (i & 1)) & 0xffffu);
    };

    // Weights: each thread some consecutive values, `each` of them.
    auto value = [](uint32_t key) __attribute__((always_inline)) {
        const uint32_t h = key & 0x8000u ? key : key ^ 0x7fffu;
        return KIND == 1 ? bf16_bits_to_f32(h) : (float)__builtin_bit_cast(_Float16, (uint16_t)h);
    };
    SampleScale& sc = rule.sc;
    uint32_t top;   // the largest value's key
    if (listed) {
        top = list[0] >> 16;
    } else {
        const uint64_t has0 = __ballot(own0 != 0), has1 = __ballot(own1 != 0);
        const int step = has0 ? __builtin_ctzll(has0) : 64 + __builtin_ctzll(has1);
        const u32x4 v = reinterpret_cast<const u32x4*>(s.bins)[64 * step + lane];
        uint32_t at = 8;
#pragma unroll
        for (int e = 3; e >= 0; --e) at = v[e] & 0xffffu ? 2 * e : v[e] >> 16 ? 2 * e + 1 : at;
        const int first_lane = __builtin_ctzll(__ballot(at < 8));
        top = 8u * (64 * step + first_lane) + lane_of(at, first_lane);
    }
    sc.m = value(top);
    const uint32_t each = (values + kSampleThreads - 1) / kSampleThreads;   // 64 at most
    uint32_t c = 0;
    uint64_t w = 0, above = 0;
    for (uint32_t i = t * each; i < min(values, (t + 1) * each); ++i) {
        const uint32_t e = entry(i);
        if (!(e & 0xffffu)) continue;
        const double y = sc.exponent(value(e >> 16));
        c += tokens_of(e);
        if (sc.in_play(y)) {
            const uint64_t one = tokens_of(e) * sc.rounded(sc.power(y, table));
            w += one;
            above += y >= rule.y_min ? one : 0ull;
        }
    }
    const bool with_min_p = rule.y_min > -INFINITY;
    if (with_min_p) {
        above = running64(above);
        if (lane == 63) atomicAdd(reinterpret_cast<unsigned long long*>(&s.above), (unsigned long long)above);
    }
    uint32_t c1 = running64(c), all;
    uint64_t w1 = running64(w), all_mass;
    if (lane == 63) s.wave32[wave] = c1, s.wave64[wave] = w1;
    __syncthreads();
    c1 += before_wave(s.wave32, wave, all);
    w1 += before_wave(s.wave64, wave, all_mass);
    const uint32_t c0 = c1 - c;
    const uint64_t w0 = w1 - w;
    above = with_min_p ? s.above : ~0ull;
    uint32_t equals = 0;
    int asked = 0;
    auto ask = [&](const SampleQuery& q, bool) -> SampleHit {
        const uint64_t owner = __ballot(c && q.at(c1, w1) && (c0 == 0 || !q.at(c0, w0)));
        SampleValues::Hit& found = s.hits[asked++];   // a place for each question: a slow wave may still read the last one's
        if (owner) {   // this wave's: that thread's values, one a lane
            const int who = __builtin_ctzll(owner);
            const uint32_t i = (64 * wave + who) * each + lane;
            const bool in = (uint32_t)lane < each && i < values;
            const uint32_t e = in ? entry(i) : 0u, mult = in ? tokens_of(e) : 0u;
            const double y = sc.exponent(value(e >> 16));
            const uint64_t one = in && sc.in_play(y) ? sc.rounded(sc.power(y, table)) : 0ull;
            const uint32_t cs = running64(mult) + lane_of(c0, who), cb = cs - mult;
            const uint64_t ws = running64(mult * one) + lane_of(w0, who), wb = ws - mult * one;
            if (mult && q.at(cs, ws) && (cb == 0 || !q.at(cb, wb))) {
                const uint32_t r = sample_among_equals(q, mult, cb, wb, one);
                found.mass = wb + r * one;
                found.key = e >> 16;
                found.rank = r;
                found.equals = mult;
            }
        }
        __syncthreads();
        equals = found.equals;
        return SampleHit{found.mass, found.key, found.rank, -1};
    };
    uint64_t kept, others = 0;
    SampleHit end;
    const SampleHit hit = rule.token(all, all_mass, above, p.u[row], kept, end, ask);
    const double fine = p.logprob ? rule.fine_tail(hit, end, top, kept, p.V) : 0.;
    if (fine != 0.) {
        for (uint32_t i = t * each; i < min(values, (t + 1) * each); ++i) {
            const uint32_t e = entry(i), key = e >> 16;
            if (!(e & 0xffffu) || key == top || (end.rank && key > end.key)) continue;
            const double y = sc.exponent(value(key));
            if (y >= rule.y_min) others += (end.rank && key == end.key ? end.rank : tokens_of(e)) * sc.fine_weight(y, table, fine);
        }
        others = running64(others);
        if (lane == 63) s.wave64[wave] = others;
    }
    __syncthreads();   // the list of values is spent
    if (fine != 0.) before_wave(s.wave64, wave, others);
    int index;
    if (equals <= kMaxTies) {
        const uint32_t bits = hit.key & 0x8000u ? hit.key : hit.key ^ 0x7fffu;
        const uint32_t want = bits | bits << 16, care = bits ? 0xffffffffu : 0x7fff7fffu;   // 0 is -0 too
        auto found = [&](int i) __attribute__((always_inline)) { s.bins[atomicAdd(&s.ties, 1u)] = (uint32_t)i; };
        auto look8 = [&](const u32x4& v, int i0) __attribute__((always_inline)) {
            uint32_t d[4];
            u16x2 least = {0xffff, 0xffff};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                d[e] = (v[e] ^ want) & care;
                least = __builtin_elementwise_min(least, __builtin_bit_cast(u16x2, d[e]));
            }
            if (least[0] && least[1]) return;
            uint32_t hits = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) hits |= (d[e] & 0xffffu ? 0u : 1u << 2 * e) | (d[e] >> 16 ? 0u : 2u << 2 * e);
            for (; hits; hits &= hits - 1) found(i0 + __builtin_ctz(hits));
        };
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            if (j * kSampleThreads >= pieces) break;
            if (t + j * kSampleThreads < pieces) look8(held[j], head + 8 * (t + j * kSampleThreads));
        }
        for (int i = t + kHeld * kSampleThreads; i < pieces; i += kSampleThreads) look8(from[i], head + 8 * i);
        if (in_head && !((first ^ want) & care & 0xffffu)) found(t);
        if (in_tail && !((last ^ want) & care & 0xffffu)) found(tail + t);
        __syncthreads();
        if ((uint32_t)t < equals) {
            const uint32_t i = s.bins[t];
            uint32_t place = 1, j = 0;
            for (; j + 4 <= equals; j += 4) {
                const u32x4 e = *reinterpret_cast<const u32x4*>(s.bins + j);
                place += (e[0] < i) + (e[1] < i) + (e[2] < i) + (e[3] < i);
            }
            for (; j < equals; ++j) place += s.bins[j] < i;
            if (place == hit.rank) s.token = (int)i;
        }
        __syncthreads();
        index = s.token;
    } else {
        __syncthreads();   // the waves' sums are read: sample_nth's memory is theirs, too
        index = sample_nth(shared.nth, x, sample_key(value(hit.key)), hit.rank);
    }
    if (t == 0) {
        p.token[row] = index;
        if (p.logprob) p.logprob[row] = fine != 0. ? rule.tail_logprob(others, fine) : rule.logprob(value(hit.key), kept);
    }
}

// Rows of more than 65535 tokens in which a count of 16 bits was too small.
template <int KIND>
__global__ __launch_bounds__(kSampleThreads) void sample_overflow_kernel(const SampleArgs p) {
    __shared__ SampleShared s;
    __shared__ double table[1 << kExpBits];
    if (p.token[blockIdx.x] == kOverflow) sample_row<KIND>(p, s, table, blockIdx.x);
}

}  // namespace sfk

static int sample_check(const sf_sample_desc* d) {
    if (!d || d->rows < 0 || d->V <= 0) return SF_EINVAL;
    if (d->dtype != SF_F32 && d->dtype != SF_BF16 && d->dtype != SF_F16) return SF_ENOTSUP;
    if (d->V > SF_SAMPLE_MAX_VOCAB || d->rows >= 1 << 22) return SF_ENOTSUP;   // a launch counts its threads in 32 bits
    return SF_OK;
}

extern "C" size_t sf_sample_workspace_bytes(const sf_sample_desc* d) {
    if (sample_check(d) != SF_OK || d->rows == 0 || sfk::sample_parts(d->rows, d->V, d->dtype) == 1) return 0;
    return (size_t)d->rows * sizeof(sfk::SampleParts);
}

extern "C" int sf_sample(const sf_sample_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = sample_check(d);
    if (st != SF_OK) return st;
    if (d->rows == 0) return SF_OK;
    if (!d->logits || !d->u || !d->token || d->ld < d->V) return SF_EINVAL;
    if (reinterpret_cast<uintptr_t>(d->logits) & (d->dtype == SF_F32 ? 3 : 1)) return SF_EINVAL;
    for (const void* q : {(const void*)d->u, (const void*)d->temperature, (const void*)d->top_k, (const void*)d->top_p,
                          (const void*)d->min_p, (const void*)d->token, (const void*)d->logprob})
        if (reinterpret_cast<uintptr_t>(q) & 3) return SF_EINVAL;
    const int parts = sfk::sample_parts(d->rows, d->V, d->dtype);
    if (parts > 1 && (!workspace || workspace_bytes < sf_sample_workspace_bytes(d))) return SF_EWORKSPACE;
    if (parts > 1 && (reinterpret_cast<uintptr_t>(workspace) & 7)) return SF_EINVAL;
    const sfk::SampleArgs p = {d->logits, d->ld, d->u, d->temperature, d->top_p, d->min_p, d->top_k, d->temperature_all, d->top_p_all,
                               d->min_p_all, d->top_k_all, d->V, d->token, d->logprob, static_cast<char*>(workspace), parts};
    const dim3 grid((unsigned)d->rows), each((unsigned)d->rows * (unsigned)parts), block(sfk::kSampleThreads);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (parts > 1) {
        hipLaunchKernelGGL(sfk::sample_parts_largest_kernel, each, block, 0, s, p);
        if (hipGetLastError() != hipSuccess) return SF_ELAUNCH;
        hipLaunchKernelGGL(sfk::sample_parts_fill_kernel, each, block, 0, s, p);
        if (hipGetLastError() != hipSuccess) return SF_ELAUNCH;
        hipLaunchKernelGGL(sfk::sample_parts_choose_kernel, grid, block, 0, s, p);
    } else if (d->dtype == SF_F32) {
        hipLaunchKernelGGL(sfk::sample_f32_kernel, grid, block, 0, s, p);
    } else {
        if (d->dtype == SF_BF16) hipLaunchKernelGGL(sfk::sample_16_kernel<1>, grid, block, 0, s, p);
        else hipLaunchKernelGGL(sfk::sample_16_kernel<2>, grid, block, 0, s, p);
        if (d->V > 65535) {
            if (hipGetLastError() != hipSuccess) return SF_ELAUNCH;
            if (d->dtype == SF_BF16) hipLaunchKernelGGL(sfk::sample_overflow_kernel<1>, grid, block, 0, s, p);
            else hipLaunchKernelGGL(sfk::sample_overflow_kernel<2>, grid, block, 0, s, p);
        }
    }
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
