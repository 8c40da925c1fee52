// block_manager.cpp -- the block manager: which pages of the KV pools are in use, and by how many sequences (host state only;
// contract in include/llmgen_host.h).  The reference's BlockManager (src/runner/block.zig) is a stack of free ids; here
// a page has a reference count, so that sequences forked from one prompt share its pages until one of them writes, and
// the free ids are an ordered set, so that the lowest go out first and a compaction has few pages to move.
#include <stdint.h>
#include <stdio.h>

#include <exception>
#include <set>
#include <unordered_map>
#include <vector>

#include "llmgen_host.h"

namespace {

struct Blocks {
    std::vector<int32_t> refs;
    std::set<int32_t> free_ids;
};

bool held(const Blocks &b, int32_t id) { return id >= 0 && (size_t)id < b.refs.size() && b.refs[id] > 0; }

// Runs f; host memory that runs out is reported and refused, not thrown through the C boundary.
template <typename F>
int guarded(const char *who, F f) {
    try {
        return f();
    } catch (const std::exception &e) {
        fprintf(stderr, "[llmgen-host] %s: %s\n", who, e.what());
        return -1;
    }
}

}  // namespace

extern "C" {

void *llmgen_blocks_create(int num_blocks) {
    if (num_blocks <= 0) return nullptr;
    Blocks *b = nullptr;
    const int rc = guarded("blocks_create", [&]() {
        b = new Blocks;
        b->refs.assign(num_blocks, 0);
        for (int32_t i = 0; i < num_blocks; ++i) b->free_ids.insert(b->free_ids.end(), i);
        return 0;
    });
    if (rc == 0) return b;
    delete b;
    return nullptr;
}

void llmgen_blocks_destroy(void *blocks) { delete static_cast<Blocks *>(blocks); }

int llmgen_blocks_free_count(const void *blocks) {
    return blocks ? (int)static_cast<const Blocks *>(blocks)->free_ids.size() : -1;
}

int llmgen_blocks_ref(const void *blocks, int id) {
    const Blocks *b = static_cast<const Blocks *>(blocks);
    return b && id >= 0 && (size_t)id < b->refs.size() ? b->refs[id] : -1;
}

int llmgen_blocks_alloc(void *blocks, int n, int32_t *out) {
    Blocks *b = static_cast<Blocks *>(blocks);
    if (!b || n < 0 || (n > 0 && !out) || (size_t)n > b->free_ids.size()) return -1;
    for (int i = 0; i < n; ++i) {
        const int32_t id = *b->free_ids.begin();
        b->free_ids.erase(b->free_ids.begin());
        b->refs[id] = 1;
        out[i] = id;
    }
    return 0;
}

int llmgen_blocks_fork(void *blocks, const int32_t *table, int n) {
    Blocks *b = static_cast<Blocks *>(blocks);
    if (!b || n < 0 || (n > 0 && !table)) return -1;
    for (int i = 0; i < n; ++i)
        if (table[i] >= 0 && !held(*b, table[i])) return -1;
    for (int i = 0; i < n; ++i)
        if (table[i] >= 0) ++b->refs[table[i]];
    return 0;
}

int llmgen_blocks_free(void *blocks, const int32_t *table, int n) {
    Blocks *b = static_cast<Blocks *>(blocks);
    if (!b || n < 0 || (n > 0 && !table)) return -1;
    return guarded("blocks_free", [&]() {
        std::unordered_map<int32_t, int32_t> drops;  // a table may name a page twice
        for (int i = 0; i < n; ++i) {
            if (table[i] < 0) continue;
            if (!held(*b, table[i]) || ++drops[table[i]] > b->refs[table[i]]) return -1;
        }
        std::set<int32_t> gone;  // made first: nothing has changed yet if memory runs out
        for (const auto &d : drops)
            if (d.second == b->refs[d.first]) gone.insert(d.first);
        for (const auto &d : drops) b->refs[d.first] -= d.second;
        b->free_ids.merge(gone);
        return 0;
    });
}

int llmgen_blocks_writable(void *blocks, int32_t *table, int idx, int32_t *src, int32_t *dst) {
    Blocks *b = static_cast<Blocks *>(blocks);
    if (!b || !table || idx < 0 || !src || !dst || !held(*b, table[idx])) return -1;
    const int32_t old = table[idx];
    if (b->refs[old] == 1) return 0;
    int32_t fresh;
    if (llmgen_blocks_alloc(blocks, 1, &fresh) != 0) return -1;
    --b->refs[old];
    table[idx] = fresh;
    *src = old;
    *dst = fresh;
    return 1;
}

int llmgen_blocks_compact(void *blocks, int32_t *src, int32_t *dst, int cap) {
    Blocks *b = static_cast<Blocks *>(blocks);
    if (!b || cap < 0 || (cap > 0 && (!src || !dst))) return -1;
    return guarded("blocks_compact", [&]() {
        // the k-th lowest free id takes the k-th highest used one, while it lies below it
        std::vector<int32_t> from, to;
        int32_t high = (int32_t)b->refs.size() - 1;
        for (int32_t id : b->free_ids) {
            while (high > id && b->refs[high] == 0) --high;
            if (high <= id) break;
            from.push_back(high--);
            to.push_back(id);
        }
        const int n = (int)from.size();
        if (n > cap) return -1;
        std::set<int32_t> freed(from.begin(), from.end());
        for (int i = 0; i < n; ++i) {
            b->refs[to[i]] = b->refs[from[i]];
            b->refs[from[i]] = 0;
            b->free_ids.erase(to[i]);
            src[i] = from[i];
            dst[i] = to[i];
        }
        b->free_ids.merge(freed);
        return n;
    });
}

int llmgen_blocks_remap(int32_t *table, int n, const int32_t *src, const int32_t *dst, int n_pairs) {
    if (n < 0 || n_pairs < 0 || (n > 0 && !table) || (n_pairs > 0 && (!src || !dst))) return -1;
    return guarded("blocks_remap", [&]() {
        std::unordered_map<int32_t, int32_t> to;
        for (int i = 0; i < n_pairs; ++i) to[src[i]] = dst[i];
        for (int i = 0; i < n; ++i) {
            if (table[i] < 0) continue;
            const auto it = to.find(table[i]);
            if (it != to.end()) table[i] = it->second;
        }
        return 0;
    });
}

}  // extern "C"
