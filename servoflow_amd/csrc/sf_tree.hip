// Trees of drafted tokens (gfx950): ancestor masks, the confirmed path, and the
// cache with that path alone.
//
// All of it is whole numbers and a few kilobytes, so each kernel is bound by its launch
// and one or two round trips to memory.  us alone, for one tree of 16 nodes over 8
// heads of 128 channels and for 32 trees of 64 over 32 heads of 64: tables 1.4 and
// 3.7, path 1.8 and 4.1, kept tokens 3.1 and 5.6 (1.6 MB read and written).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sf_hip.h"
#include "sf_kv4.h"

namespace sfk {

// One thread for each word of a node's mask: it walks the node's ancestors in LDS, whose
// indices fall at every step, so a walk ends whatever the parents hold.  (A chain of T nodes
// takes T steps of an LDS read each.)
__global__ __launch_bounds__(256) void tree_build_kernel(const int32_t* parents, int T, int words, uint32_t* masks,
                                                         int32_t* depth) {
    __shared__ int up[SF_TREE_MAX_NODES];
    const int64_t b = blockIdx.y;
    for (int i = threadIdx.x; i < T; i += 256) up[i] = parents[b * T + i];
    __syncthreads();
    const int at = blockIdx.x * 256 + threadIdx.x;
    if (at >= T * words) return;
    const int node = at / words, word = at % words;
    uint32_t m = 0;
    int n = 0;
    for (int j = node;; ++n) {
        if (j >> 5 == word) m |= 1u << (j & 31);
        const int p = up[j];
        if (p < 0 || p >= j) break;
        j = p;
    }
    masks[b * T * words + at] = m;
    if (word == 0) depth[b * T + node] = n;
}

// One wave for each batch element: a step looks at every node behind the current one
// for a child with the sampled token, 64 at a time from the words behind it.
__global__ __launch_bounds__(64) void tree_accept_kernel(const int32_t* parents, int64_t tree_stride, const int32_t* drafted,
                                                         const int32_t* sampled, int T, int32_t* nodes, int32_t* count,
                                                         int32_t* tokens) {
    __shared__ int up[SF_TREE_MAX_NODES], draft[SF_TREE_MAX_NODES], drawn[SF_TREE_MAX_NODES];
    const int64_t b = blockIdx.x;
    const int lane = threadIdx.x;
    for (int i = lane; i < T; i += 64) {
        up[i] = parents[b * tree_stride + i];
        draft[i] = drafted[b * T + i];
        drawn[i] = sampled[b * T + i];
    }
    __syncthreads();
    int cur = 0, n = 0;
    while (true) {
        const int token = drawn[cur];
        if (lane == 0) nodes[b * T + n] = cur, tokens[b * T + n] = token;
        ++n;
        int next = -1;
        for (int base = cur + 1; base < T && next < 0; base += 64) {
            const int j = base + lane;
            const uint64_t hit = __ballot(j < T && up[min(j, T - 1)] == cur && draft[min(j, T - 1)] == token);
            if (hit) next = base + __builtin_ctzll(hit);
        }
        if (next < 0) break;   // next > cur: T steps at most
        cur = next;
    }
    for (int i = n + lane; i < T; i += 64) nodes[b * T + i] = tokens[b * T + i] = -1;
    if (lane == 0) count[b] = n;
}

// A workgroup for each batch element, head and part of its tokens (key codes, value
// codes, parameters: bytes of their own, so the parts need not meet; of one token they are too
// few for a workgroup, and three parts run side by side).  Every moved
// token is read into LDS before the first is written.
template <int D>
__global__ __launch_bounds__(256) void kv4_keep_kernel(uint8_t* cache, int H, int capacity, int64_t blocks, const int32_t* nodes,
                                                       int n, const int32_t* first) {
    constexpr int U = D / 8;   // dwords of key codes of a token, and of value codes; parameters are D / 32
    extern __shared__ uint32_t held[];
    __shared__ int from[SF_TREE_MAX_NODES], last;
    const int part = blockIdx.x % 3, h = blockIdx.x / 3;
    const int64_t b = blockIdx.y;
    uint8_t* base = cache + (b * H + h) * blocks * Kv4<D>::kBytes;
    const int at0 = first[b];
    if (threadIdx.x == 0) last = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        const int64_t src = (int64_t)at0 + nodes[b * n + i], dst = (int64_t)at0 + i;
        const bool move = nodes[b * n + i] >= 0 && src != dst && src >= 0 && src < capacity && dst >= 0 && dst < capacity;
        from[i] = move ? (int)src : -1;
        if (move) atomicMax(&last, i + 1);
    }
    __syncthreads();
    const int m = last;
    auto block = [&](int slot) { return base + (int64_t)(slot / kKvBlock) * Kv4<D>::kBytes; };
    auto par = [](int tok, int u) {   // u: key groups, then value groups
        return u < D / 64 ? Kv4<D>::key_par(tok, u) : Kv4<D>::value_par(tok, u - D / 64);
    };
    if (part == 0) {
        for (int i = threadIdx.x; i < m * U; i += 256) {
            const int src = from[i / U];
            if (src >= 0) held[i] = *reinterpret_cast<const uint32_t*>(block(src) + Kv4<D>::key_dword(src % kKvBlock, i % U));
        }
        __syncthreads();
        for (int i = threadIdx.x; i < m * U; i += 256) {
            const int dst = at0 + i / U;
            if (from[i / U] >= 0) *reinterpret_cast<uint32_t*>(block(dst) + Kv4<D>::key_dword(dst % kKvBlock, i % U)) = held[i];
        }
    } else if (part == 1) {   // single bytes, D / 2 of them
        constexpr int N = D / 2;
        uint8_t* bytes = reinterpret_cast<uint8_t*>(held);
        for (int i = threadIdx.x; i < m * N; i += 256) {
            const int src = from[i / N], v = i % N;
            if (src >= 0) bytes[i] = block(src)[Kv4<D>::kV + Kv4<D>::value_byte(src % kKvBlock, v >> 4, v & 15)];
        }
        __syncthreads();
        for (int i = threadIdx.x; i < m * N; i += 256) {
            const int dst = at0 + i / N, v = i % N;
            if (from[i / N] >= 0) block(dst)[Kv4<D>::kV + Kv4<D>::value_byte(dst % kKvBlock, v >> 4, v & 15)] = bytes[i];
        }
    } else {
        constexpr int N = D / 32;
        for (int i = threadIdx.x; i < m * N; i += 256) {
            const int src = from[i / N];
            if (src >= 0) held[i] = *reinterpret_cast<const uint32_t*>(block(src) + par(src % kKvBlock, i % N));
        }
        __syncthreads();
        for (int i = threadIdx.x; i < m * N; i += 256) {
            const int dst = at0 + i / N;
            if (from[i / N] >= 0) *reinterpret_cast<uint32_t*>(block(dst) + par(dst % kKvBlock, i % N)) = held[i];
        }
    }
}

}  // namespace sfk

static inline bool tree_aligned(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

extern "C" int sf_tree_build(const int32_t* parents, int32_t trees, int32_t T, uint32_t* masks, int32_t* depth, void* stream) {
    if (trees < 0 || T <= 0) return SF_EINVAL;
    if (T > SF_TREE_MAX_NODES || trees > 65535) return SF_ENOTSUP;   // the grid's second dimension
    if (trees == 0) return SF_OK;
    if (!tree_aligned(parents) || !tree_aligned(masks) || !tree_aligned(depth)) return SF_EINVAL;
    const int words = (T + 31) / 32;
    hipLaunchKernelGGL(sfk::tree_build_kernel, dim3((unsigned)(T * words + 255) / 256, (unsigned)trees), dim3(256), 0,
                       static_cast<hipStream_t>(stream), parents, T, words, masks, depth);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}

extern "C" int sf_tree_accept(const int32_t* parents, int32_t each, const int32_t* drafted, const int32_t* sampled, int32_t B,
                              int32_t T, int32_t* nodes, int32_t* count, int32_t* tokens, void* stream) {
    if (B < 0 || T <= 0) return SF_EINVAL;
    if (T > SF_TREE_MAX_NODES || B >= 1 << 24) return SF_ENOTSUP;   // a launch counts its threads in 32 bits
    if (B == 0) return SF_OK;
    for (const void* p : {(const void*)parents, (const void*)drafted, (const void*)sampled, (const void*)nodes,
                          (const void*)count, (const void*)tokens})
        if (!tree_aligned(p)) return SF_EINVAL;
    hipLaunchKernelGGL(sfk::tree_accept_kernel, dim3((unsigned)B), dim3(64), 0, static_cast<hipStream_t>(stream), parents,
                       each ? (int64_t)T : 0, drafted, sampled, T, nodes, count, tokens);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}

extern "C" int sf_kv4_keep(const sf_kv4_cache* cache, const int32_t* nodes, int32_t n, const int32_t* first, void* stream) {
    if (!cache || cache->B <= 0 || cache->H <= 0 || cache->capacity <= 0 || n < 0) return SF_EINVAL;
    if ((cache->D != 64 && cache->D != 128) || n > SF_TREE_MAX_NODES) return SF_ENOTSUP;
    // the grid's second dimension; a launch counts its threads in 32 bits
    if (cache->B > 65535 || cache->H > 65535 || (int64_t)cache->B * cache->H >= 1 << 22) return SF_ENOTSUP;
    if (n == 0) return SF_OK;
    if (!cache->data || (reinterpret_cast<uintptr_t>(cache->data) & 15) || !tree_aligned(nodes) || !tree_aligned(first))
        return SF_EINVAL;
    const dim3 grid(3u * (unsigned)cache->H, (unsigned)cache->B);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const unsigned lds = (unsigned)n * (unsigned)cache->D / 2;   // 64 KB at most
    uint8_t* data = static_cast<uint8_t*>(cache->data);
    const int64_t blocks = sfk::kv4_blocks(cache->capacity);
    if (cache->D == 64) hipLaunchKernelGGL(sfk::kv4_keep_kernel<64>, grid, dim3(256), lds, s, data, cache->H, cache->capacity, blocks, nodes, n, first);
    else hipLaunchKernelGGL(sfk::kv4_keep_kernel<128>, grid, dim3(256), lds, s, data, cache->H, cache->capacity, blocks, nodes, n, first);
    return hipGetLastError() == hipSuccess ? SF_OK : SF_ELAUNCH;
}
