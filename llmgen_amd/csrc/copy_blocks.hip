// copy_blocks.hip -- copies of pages inside the KV pools (hip_copy_blocks, include/llmgen_cache.h).
//
// A fork or a compaction moves the same pages in the K and V pools of every layer, so one launch takes a table of pools
// times a table of pairs, both in the kernel's arguments: nothing is uploaded, and a captured launch keeps its tables.
// Pure HBM copy: the 16-byte pieces of all the launch's pages stand in one row, LOADS of them a thread, so that no thread
// idles whatever the page size (pages of 1088 bytes 144 -> 74 us against a workgroup a page; of 8704 bytes 206 -> 210 us).
// A thread's loads are issued before its stores, both past the caches (8704 bytes: 232 -> 210 us).  The pairs have no
// order (the host refuses chains), so neither do the workgroups.  1096 pages of 8704 bytes in 56 pools: 193 to 210 us (box to
// box), 5.1 to 5.5 TB/s.
#include "cache_common.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {

using llmgen_cache::page_div;
using llmgen_cache::PageDiv;
using llmgen_cache::refuse;

constexpr int MAX_POOLS = 64, MAX_PAIRS = 256;  // one launch's tables: 512 + 2048 bytes of arguments
constexpr int THREADS = 512, LOADS = 2;

struct Copies {
    char *pool[MAX_POOLS];
    int src[MAX_PAIRS], dst[MAX_PAIRS];
};

__device__ __forceinline__ u32x4_t take(const char *p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(p));
}
__device__ __forceinline__ void put(char *p, u32x4_t x) {
    __builtin_nontemporal_store(x, reinterpret_cast<u32x4_t *>(p));
}

__global__ void __launch_bounds__(THREADS) copy_blocks_kernel(const Copies c, PageDiv per_pool, PageDiv per_page,
                                                              int total) {
    const char *src[LOADS];
    char *dst[LOADS];
    u32x4_t x[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int at = ((int)blockIdx.x * LOADS + i) * THREADS + (int)threadIdx.x;
        src[i] = nullptr;
        if (at >= total) continue;
        const int page = per_page(at), pair = per_pool(page);
        char *pool = c.pool[page - pair * per_pool.bs] + (long)(at - page * per_page.bs) * 16;
        const long block_bytes = (long)per_page.bs * 16;
        src[i] = pool + c.src[pair] * block_bytes;
        dst[i] = pool + c.dst[pair] * block_bytes;
        x[i] = take(src[i]);
    }
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
        if (src[i]) put(dst[i], x[i]);
}

// Every id in range, no page written twice, none both read and written.
bool independent(const int32_t *src, const int32_t *dst, int n, int num_blocks) {
    std::vector<int32_t> written, read;
    written.reserve(n);
    read.reserve(n);
    for (int i = 0; i < n; ++i) {
        if (src[i] < 0 || src[i] >= num_blocks || dst[i] < 0 || dst[i] >= num_blocks) return false;
        if (src[i] == dst[i]) continue;
        written.push_back(dst[i]);
        read.push_back(src[i]);
    }
    std::sort(written.begin(), written.end());
    if (std::adjacent_find(written.begin(), written.end()) != written.end()) return false;
    for (int32_t r : read)
        if (std::binary_search(written.begin(), written.end(), r)) return false;
    return true;
}

}  // namespace

extern "C" void hip_copy_blocks(void *const *pools, int n_pools, size_t block_bytes, int num_blocks, const int32_t *src,
                                const int32_t *dst, int n) {
    const char *who = "copy_blocks";
    if (n <= 0 || n_pools <= 0) return;
    if (!pools || !src || !dst || num_blocks <= 0) {
        refuse(who, "a table is missing, or there are no pages");
        return;
    }
    if (block_bytes == 0 || block_bytes % 16 != 0 || block_bytes > (size_t)1 << 28) {
        refuse(who, "the page size must be a multiple of 16 bytes, at most 256 MiB");
        return;
    }
    for (int i = 0; i < n_pools; ++i)
        if (!pools[i] || ((uintptr_t)pools[i] & 15)) {
            refuse(who, "a pool is missing or not 16-byte aligned");
            return;
        }
    try {
        if (!independent(src, dst, n, num_blocks)) {
            refuse(who, "page ids out of range, a page written twice, or one both read and written");
            return;
        }
    } catch (const std::bad_alloc &) {
        refuse(who, "out of host memory");
        return;
    }
    const int pieces = (int)(block_bytes / 16);
    Copies c;
    int pairs = 0;
    auto flush = [&]() {
        for (int p0 = 0; p0 < n_pools; p0 += MAX_POOLS) {
            const int m = std::min(n_pools - p0, MAX_POOLS);
            for (int i = 0; i < m; ++i) c.pool[i] = static_cast<char *>(pools[p0 + i]);
            const int total = pieces * m * pairs;
            hipLaunchKernelGGL(copy_blocks_kernel, dim3((total + THREADS * LOADS - 1) / (THREADS * LOADS)), dim3(THREADS), 0,
                               g_llmgen_stream, c, page_div(m), page_div(pieces), total);
        }
        pairs = 0;
    };
    // a launch's pieces are counted in 30 bits
    const long per_launch = std::min<long>(MAX_PAIRS, (1L << 30) / ((long)pieces * std::min(n_pools, MAX_POOLS)));
    for (int i = 0; i < n; ++i) {
        if (src[i] == dst[i]) continue;
        c.src[pairs] = src[i];
        c.dst[pairs] = dst[i];
        if (++pairs == per_launch) flush();
    }
    if (pairs) flush();
}
