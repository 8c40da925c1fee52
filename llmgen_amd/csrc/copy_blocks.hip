// copy_blocks.hip -- copies of pages inside the KV pools (hip_copy_blocks, include/llmgen_cache.h).
//
// A fork or a compaction moves the same pages in the K and V pools of every layer, so one launch takes a table of pools
// times a table of pairs, both in the kernel's arguments: nothing is uploaded, and a captured launch keeps its tables.
// Pure HBM copy: a workgroup moves CHUNK bytes with 16-byte accesses, all of a thread's loads issued before its stores.
// The pairs have no order (the host refuses chains), so neither do the workgroups.
#include "cache_common.h"

#include <algorithm>
#include <new>
#include <vector>

namespace {

using llmgen_cache::refuse;

constexpr int MAX_POOLS = 64, MAX_PAIRS = 256;  // one launch's tables: 512 + 2048 bytes of arguments
constexpr int THREADS = 256, LOADS = 4, CHUNK = THREADS * LOADS * 16;

struct Copies {
    char *pool[MAX_POOLS];
    int src[MAX_PAIRS], dst[MAX_PAIRS];
};

__global__ void __launch_bounds__(THREADS) copy_blocks_kernel(const Copies c, int n_pools, int chunks, long block_bytes) {
    const int chunk = blockIdx.x % chunks;
    const int rest = blockIdx.x / chunks, pair = rest / n_pools;
    char *pool = c.pool[rest % n_pools];
    const char *src = pool + c.src[pair] * block_bytes;
    char *dst = pool + c.dst[pair] * block_bytes;
    const long at = (long)chunk * CHUNK + threadIdx.x * 16;
    u32x4_t x[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
        if (at + i * THREADS * 16 < block_bytes) x[i] = ld16(src + at + i * THREADS * 16);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
        if (at + i * THREADS * 16 < block_bytes) *reinterpret_cast<u32x4_t *>(dst + at + i * THREADS * 16) = x[i];
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
    if (block_bytes == 0 || block_bytes % 16 != 0 || block_bytes > (size_t)1 << 40) {
        refuse(who, "the page size must be a multiple of 16 bytes");
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
    const long chunks = ((long)block_bytes + CHUNK - 1) / CHUNK;
    Copies c;
    int pairs = 0;
    auto flush = [&]() {
        for (int p0 = 0; p0 < n_pools; p0 += MAX_POOLS) {
            const int m = std::min(n_pools - p0, MAX_POOLS);
            for (int i = 0; i < m; ++i) c.pool[i] = static_cast<char *>(pools[p0 + i]);
            hipLaunchKernelGGL(copy_blocks_kernel, dim3((unsigned)(chunks * m * pairs)), dim3(THREADS), 0, g_llmgen_stream,
                               c, m, (int)chunks, (long)block_bytes);
        }
        pairs = 0;
    };
    // chunks * pools * pairs of one launch must fit the grid
    const long per_launch = std::max(1L, std::min<long>(MAX_PAIRS, 0x7fffffffL / (chunks * std::min(n_pools, MAX_POOLS))));
    for (int i = 0; i < n; ++i) {
        if (src[i] == dst[i]) continue;
        c.src[pairs] = src[i];
        c.dst[pairs] = dst[i];
        if (++pairs == per_launch) flush();
    }
    if (pairs) flush();
}
