// window.hip -- attention with a sliding window and sinks over bf16 pages, and causal prefill over 4-bit pages with or
// without them (gfx950; contracts in include/llmgen_cache.h).
//
// A row at position p sees keys k <= p with k > p - window or k < sinks; without a window that is plain causal
// attention.  What bounds these kernels is what bounds attention over the whole context -- HBM for one query row a
// sequence, the matrix cores for many -- so they are built from the same workgroups, and the work they save is the keys
// they do not walk: a decode row reads window + sinks keys whatever its context, and a query tile of 64 rows walks the
// 64-key tiles of the sinks and of its own window, of which only those cut by an end of either, or by the diagonal, pay
// for masks.
//   * decode over bf16 pages: the split-K workgroup of decode_kernel.h, walking the visible keys only;
//   * prefill: the workgroup of window_kernel.h.  A unit is a query tile x KV head x group of NW / 2 heads; with few
//     units each one's key tiles are split over up to 64 workgroups, whose partial (m, l, O) the last to finish merge in
//     order out of the caller's scratch;
//   * 4-bit pages: a tile's codes are loaded a tile ahead into registers (one 16-byte run of 32 codes of K and one of V
//     a thread) and converted to bf16 on the way into LDS, so the products and the softmax are the same code;
//   * single rows of a prefill step are streamed by a decode launch before it, in the same scratch.
// Measured: decode of 64 sequences x 8 KV heads with 4096 visible keys each (1.01 GB) 166 us, 6.1 TB/s; of one sequence
// with 1000 visible keys 7.7 us, launch, split and merge.  Prefill of 16384 rows x 32 heads with a window of 1024 keys
// (267 GFLOP) 338 us, 790 TFLOP/s; of 8192 rows x 32 heads on 4-bit pages without one (550 GFLOP) 545 us, 1010 TFLOP/s,
// bound by the softmax's vector instructions, which the two workgroups of a CU run beside each other's products.
#include "cache_common.h"
#include "decode_kernel.h"
#include "hip_common.h"
#include "window_kernel.h"

#include <algorithm>

namespace {

using llmgen_cache::check_attention;
using llmgen_cache::NO_WINDOW;
using llmgen_cache::refuse;
using llmgen_cache::split_work;
using llmgen_cache::Work;
using llmgen_cache::WORK_COUNTERS;

// ------------------------------------------------------------------------------------------------------------
// Decode over bf16 pages
// ------------------------------------------------------------------------------------------------------------
struct RowArgs {
    bf16_t *out;
    const bf16_t *q, *kc, *vc;
    const int *bt, *ctx, *cu_q, *tile_seq;
    int S, nq, nkv, max_blocks, block_size, bs_shift;
    float sl2;
    int window, sinks, span = 0, nparts = 1;
    float *part_o = nullptr, *part_ml = nullptr;
    int *counters = nullptr;
};

template <int G, int NT, bool POW2, int W>
__global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(G == 4 && W == 8 ? 2 : 3)))
    attn_decode_window_kernel(const RowArgs a) {
    using namespace llmgen_decode;
    __shared__ __attribute__((aligned(16))) unsigned char lds[sizeof(DecodeLds<G, NT, W>)];
    const int kvh = blockIdx.x % a.nkv;
    const long rest = blockIdx.x / a.nkv;
    decode_split_body<G, NT, POW2, false, W, true>(
        a.out, a.part_o, a.part_ml, a.q, a.kc, a.vc, a.bt, a.ctx, a.nq, a.nkv, a.max_blocks, a.block_size, a.bs_shift,
        a.sl2, a.span, a.nparts, a.nparts, a.counters, a.cu_q, a.tile_seq, nullptr, nullptr, nullptr, nullptr, nullptr,
        kvh, (int)(rest % a.S), (int)(rest / a.S), a.S, lds, a.window, a.sinks);
}

template <int G, int NT, int W>
void launch_rows(const RowArgs &a) {
    auto kern = a.bs_shift >= 0 ? attn_decode_window_kernel<G, NT, true, W> : attn_decode_window_kernel<G, NT, false, W>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((long)a.nkv * a.S * a.nparts)), dim3(64 * W), 0, g_llmgen_stream, a);
}

void launch_rows_g(const RowArgs &a, int waves) {
    switch (a.nq / a.nkv) {
        case 1: waves == 8 ? launch_rows<1, 2, 8>(a) : launch_rows<1, 2, 4>(a); break;
        case 2: waves == 8 ? launch_rows<2, 2, 8>(a) : launch_rows<2, 2, 4>(a); break;
        case 4: waves == 8 ? launch_rows<4, 2, 8>(a) : launch_rows<4, 2, 4>(a); break;
        case 8: launch_rows<8, 2, 4>(a); break;
        default: launch_rows<16, 1, 4>(a); break;
    }
}

// The launch over a.S sequences (or entries of a tile list, `rows` of which have a single row) of up to max_ctx keys;
// false if the grid would be too large.
bool launch_split_rows(RowArgs a, int rows, int max_ctx, const Work &w) {
    const int G = a.nq / a.nkv;
    // How the keys are split, measured over 1 to 64 sequences x 8 KV heads of 300 to 8000 visible keys:
    //   * G = 4, whose 8-wave workgroup fills a CU: always 8 waves, and as many spans as there are CUs for (8 sequences of
    //     4096 keys: 4 spans of 8 waves 30.7 us, 8 of 4 waves 55 us), but no two of up to 1024 keys in all (16 sequences of
    //     700 keys: 15.9 us whole, 20.5 us in two);
    //   * G <= 2: one span for a CU or more a pair, of 8 waves, or of 4 for two pairs a CU (64 sequences of 300 keys 16.3
    //     and 20.0 us); from half a pair a CU on one of 8 up to 1024 keys (24 sequences of 700: 16.0 us, four of 4 waves
    //     20.0 us), above that four of 4 (24 of 4096: 68.9 us, one of 8 73.6 us, two of 8 84.9 us); fewer pairs: spans
    //     of 4 waves, at least a round each, up to 8 of them, or 16 below a quarter of a pair a CU (8 sequences of 4096
    //     keys: 8 spans 28.2 us, 4 of 8 waves 29.5 us); below an eighth 16 or more of 8 waves where 16 of 4 would be longer
    //     than a round (one sequence of 8000 keys: 16 of 8 waves 13.9 us, 16 of 4 waves 15.7 us, 64 17.9 us);
    //   * G >= 8: 4 waves, up to two workgroups a CU, and up to 16 spans (one sequence of 8000 keys: 16 spans 21.8 us, 64
    //     35 us), one up to 384 keys from a quarter of a pair a CU on (16 sequences of 300: 10.7 us, three 14.6 us).
    const long pairs = (long)rows * a.nkv, cus = llmgen_num_cus(), wtok = G >= 16 ? 16 : 32;
    long keys = std::max(1, std::min(max_ctx, a.max_blocks * a.block_size));
    keys = std::min(keys, (long)a.window + a.sinks + wtok + 4);
    const long rounds4 = (keys + 4 * wtok - 1) / (4 * wtok), rounds8 = (keys + 8 * wtok - 1) / (8 * wtok);
    int waves = 4;
    long parts = 1;
    if (G == 4) {
        waves = 8;
        parts = std::min(std::max(cus / pairs, 1L), rounds8);
        if (parts == 2 && keys <= 1024) parts = 1;
    } else if (G <= 2) {
        if (pairs * 2 >= cus) {
            if (pairs < cus && keys > 1024) parts = 4;
            else if (pairs < 2 * cus) waves = 8;
        } else if (pairs * 8 >= cus || rounds4 <= 16) {
            parts = std::min(rounds4, pairs * 4 >= cus ? 8L : 16L);
        } else {
            waves = 8;
            parts = std::min({rounds8, cus / pairs, std::max(16L, rounds8 / 2)});
        }
    } else if (keys > 384 || pairs * 4 < cus) {
        parts = std::min({(2 * cus + pairs - 1) / pairs, rounds4, std::max(16L, rounds4 / 8)});
    }
    parts = std::min<long>({parts, 256, w.floats / ((long)a.S * a.nq * (llmgen_decode::HD + 2))});
    if (parts < 1 || (long)a.S * a.nkv > WORK_COUNTERS) parts = 1;
    if ((long)a.S * a.nkv * parts > 0x7fffffffL) return false;
    a.span = (int)(((keys + parts - 1) / parts + wtok - 1) / wtok * wtok);
    a.nparts = (int)parts;
    if (parts > 1) {
        a.part_o = w.part;
        a.part_ml = w.part + (long)a.S * a.nq * parts * llmgen_decode::HD;
        a.counters = w.counters;
    }
    launch_rows_g(a, waves);
    return true;
}

// ------------------------------------------------------------------------------------------------------------
// Prefill
// ------------------------------------------------------------------------------------------------------------
// Pieces a unit, and key tiles a piece has at least: 4 up to 16 pieces, 8 beyond.  5 rows behind 32768 keys, 8 units: 70
// us with 16 pieces and 35.2 us with 64 on 4-bit pages, 73 and 38.4 us on bf16 ones; 100 rows behind 8000 keys, 16 units,
// 126 tiles: 32.8 us with 16 pieces, 37.1 us with 32, 42.5 us with 8.
constexpr int PIECES_MAX = 64, PIECE_MIN_TILES = 4, UNIT_COUNTERS = 9;  // a counter for each group of pieces, one for those

template <int NW, int MODE>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2)))
    attn_prefill_window_kernel(const llmgen_window::WindowArgs a, int n_split, int P, float *__restrict__ part,
                               int *__restrict__ counters) {
    using namespace llmgen_window;
    __shared__ __attribute__((aligned(16))) unsigned char lds[sizeof(WindowLds<NW>)];
    __shared__ int s_last;
    // the first n_split units (the last tiles of the list) have P workgroups each, the others one
    const int bid = (int)blockIdx.x;
    const bool split = bid < n_split * P;
    const int unit = split ? bid % n_split : bid - n_split * (P - 1), piece = split ? bid / n_split : 0;
    int pe = 1, j0 = 0, j1 = -1;
    constexpr int PSTRIDE = NW * PART_WAVE_FLOATS;
    float *base = nullptr;
    if (NW <= 4 && split) {  // which share of the unit's key tiles
        const int tile = a.n_tiles - 1 - unit / (a.nkv * a.head_groups);
        const int s = a.tile_seq[tile], q0 = a.tile_q0[tile], q_len = a.cu_q[s + 1] - a.cu_q[s];
        const int ctx = (int)min((long)a.ctx_lens[s], (long)a.max_blocks * a.div.bs);
        const int n = (q_len > 1 || a.single) && ctx >= q_len
                          ? key_tiles(ctx - q_len + q0, ctx - q_len + min(q0 + BQ, q_len), a.window, a.sinks).n
                          : 0;
        pe = n < 2 ? 1 : min(min(P, (n + PIECE_MIN_TILES - 1) / PIECE_MIN_TILES), max(16, n / 8));
        if (piece >= pe) return;
        if (pe > 1) {
            base = part + (long)unit * P * PSTRIDE;
            j0 = (int)((long)piece * n / pe);
            j1 = (int)((long)(piece + 1) * n / pe);
        }
    }
    float *mine = base ? base + (long)piece * PSTRIDE : nullptr;
    window_body<NW, MODE>(a, unit, lds, j0, j1, mine);
    if constexpr (NW <= 4) {
        // The last of the pieces to finish merges them, up to FAN; of more, the last of each 4 or FAN neighbours merges
        // these, and the last of the mergers their results: a CU reads 66 KB a piece (100 rows behind 8000 keys in 16
        // pieces: 31.8 us in one go, 26.8 us in two; 64 rows behind 1000 keys in 5 pieces: 18.8 us in one go, 21.5 us in
        // two).
        int *cnt = counters + unit * UNIT_COUNTERS;
        const int fan = pe > FAN && pe <= 16 ? 4 : FAN;
        for (int at = piece, n = pe, step = 1; n > 1; step *= fan) {
            // publish (device-coherent stores, complete before the barrier), then draw a ticket
            const int g = at / fan, first = g * fan, of = min(fan, n - first);
            float *parts = base + (long)first * step * PSTRIDE;
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (threadIdx.x == 0)
                s_last = __hip_atomic_fetch_add(cnt + g, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
            __syncthreads();
            if (!s_last) return;
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
            merge_parts<NW>(a, unit, parts, step * PSTRIDE * (int)sizeof(float), of, n > fan ? parts : nullptr);
            if (threadIdx.x == 0) __hip_atomic_store(cnt + g, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            at = g;
            n = (n + fan - 1) / fan;
            cnt += UNIT_COUNTERS - 1;
        }
    }
}

template <int NW>
void launch_prefill(int mode, const llmgen_window::WindowArgs &a, long units, long n_split, int P, const Work &w) {
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned)(units + n_split * (P - 1))), dim3(64 * NW), 0, g_llmgen_stream, a,
                           (int)n_split, P, w.part, w.counters);
    };
    using namespace llmgen_window;
    if constexpr (NW <= 4) {
        if (mode == KV4) return go(attn_prefill_window_kernel<NW, KV4>);
    }
    if (mode == DMA_BLOCK) go(attn_prefill_window_kernel<NW, DMA_BLOCK>);
    else if (mode == DMA_ROW4) go(attn_prefill_window_kernel<NW, DMA_ROW4>);
    else go(attn_prefill_window_kernel<NW, DMA_FLAT>);
}

void prefill(const char *who, bool kv4, bf16_t *out, const bf16_t *q, const void *kc, const void *vc, const int *bt,
             const int *ctx, const int *cu_q, const int *tile_seq, const int *tile_q0, int n_tiles, int nq, int nkv,
             int hd, int max_blocks, int block_size, float scale, int window, int sinks, int single_rows, void *work,
             size_t work_bytes) {
    if (n_tiles <= 0 || !check_attention(who, out, q, kc, vc, bt, ctx, nq, nkv, hd, max_blocks, block_size, scale, window,
                                         sinks, work))
        return;
    if (!cu_q || !tile_seq || !tile_q0) {
        refuse(who, "a tensor is missing");
        return;
    }
    const int G = nq / nkv;
    const int bs_shift = (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1;
    const float sl2 = scale * LLMGEN_LOG2E;
    window = window ? std::min(window, NO_WINDOW) : NO_WINDOW;
    sinks = std::min(sinks, NO_WINDOW);
    using namespace llmgen_window;
    const int mode = kv4 ? KV4
                   : bs_shift >= 0 && block_size % BK == 0 ? (int)DMA_BLOCK
                   : block_size % 4 == 0                   ? (int)DMA_ROW4
                                                           : (int)DMA_FLAT;
    // one head a 2-wave workgroup at G = 1, two a 4-wave one, four an 8-wave one
    const Work w = split_work(work, work_bytes);
    // Single rows leave at once; llmgen_fill_meta puts them first in the list, which the grid walks from its end, so the
    // units before them are the ones that may be split (in another order, or with a wrong count, other units are: the
    // result is the same).
    const int rows = std::max(0, std::min(single_rows, n_tiles)), busy_tiles = n_tiles - rows;
    int nw = G == 1 ? 2 : 4;
    long units = (long)n_tiles * nkv * (G / (nw / 2));
    const long busy = (long)busy_tiles * nkv * (G / (nw / 2));
    const long slots = (long)llmgen_num_cus() * (8 / nw);  // workgroups the chip holds at once
    long P = 1;
    if (busy > 0 && busy * 2 <= slots && busy * UNIT_COUNTERS <= WORK_COUNTERS)
        P = std::min<long>({PIECES_MAX, slots / busy, w.floats / (busy * nw * PART_WAVE_FLOATS)});
    if (P < 1) P = 1;
    // bf16 pages: four heads a workgroup read each K/V tile once for all of them, two heads leave two workgroups a CU that
    // hide each other's start and end: 16384 rows x 32 heads with a window of 256 keys 186 -> 161 us with two, of 1024
    // 333 -> 321 us, of 4096 901 -> 922 us (pages whose tiles take several DMA descriptors: 177 -> 167, 342 -> 353 us).
    // Steps of at most one four-head unit a CU want the smaller ones too (a prompt of 2048 tokens 59.0 -> 51.6 us).  4-bit
    // pages, whose conversion is shared in the same way, gain more from a second workgroup: 8192 rows 555 -> 532 us.
    const int short_window = mode == DMA_ROW4 || mode == DMA_FLAT ? 512 : 2048;
    if (!kv4 && P == 1 && G >= 4 && window > short_window && (long)busy_tiles * nkv * (G / 4) > llmgen_num_cus()) {
        nw = 8;
        units = (long)n_tiles * nkv * (G / 4);
    }
    const long n_split = P > 1 ? busy : 0;
    if (units + n_split * (P - 1) > 0x7fffffffL || (long)n_tiles * nkv > 0x7fffffffL) {
        refuse(who, "too many tiles");
        return;
    }
    if (single_rows != 0) {
        // split as a decode launch's rows are, in the scratch that the second launch uses after it
        const int known = single_rows > 0 ? rows : n_tiles;
        const bool ok = kv4 ? llmgen_kv4_rows_of_prefill(out, q, static_cast<const uint8_t *>(kc),
                                                         static_cast<const uint8_t *>(vc), bt, ctx, cu_q, tile_seq, n_tiles,
                                                         known, nq, nkv, max_blocks, block_size, sl2, window, sinks, work,
                                                         work_bytes)
                            : launch_split_rows(RowArgs{out, q, static_cast<const bf16_t *>(kc),
                                                        static_cast<const bf16_t *>(vc), bt, ctx, cu_q, tile_seq, n_tiles,
                                                        nq, nkv, max_blocks, block_size, bs_shift, sl2, window, sinks},
                                                known, max_blocks * block_size, w);
        if (!ok) {
            refuse(who, "too many tiles");
            return;
        }
    }
    const WindowArgs a{out, q, kc, vc, bt, ctx, cu_q, tile_seq, tile_q0, n_tiles, nq, nkv, G, G / (nw / 2), max_blocks,
                       llmgen_cache::page_div(block_size), sl2, window, sinks, single_rows == 0};
    if (nw == 2) launch_prefill<2>(mode, a, units, n_split, (int)P, w);
    else if (nw == 4) launch_prefill<4>(mode, a, units, n_split, (int)P, w);
    else launch_prefill<8>(mode, a, units, 0, 1, w);
}

__global__ void __launch_bounds__(256) clear_counters_kernel(int *counters, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) counters[i] = 0;
}

}  // namespace

extern "C" size_t hip_attn_work_bytes(void) {
    // counters, and room for 512 partial results of 4-wave prefill workgroups (or 66,000 of decode rows)
    return llmgen_cache::WORK_HEAD + (size_t)512 * llmgen_prefill::PART_FLOATS * sizeof(float);
}

extern "C" void hip_attn_work_init(void *work, size_t work_bytes) {
    if (!work || ((uintptr_t)work & 15)) {
        refuse("attn_work_init", "the scratch must be 16-byte aligned device memory");
        return;
    }
    const int n = (int)std::min<size_t>(work_bytes / sizeof(int), WORK_COUNTERS);
    if (n <= 0) return;
    hipLaunchKernelGGL(clear_counters_kernel, dim3((n + 255) / 256), dim3(256), 0, g_llmgen_stream,
                       static_cast<int *>(work), n);
}

extern "C" void hip_attn_decode_window(bf16_t *out, const bf16_t *q, const bf16_t *k_cache, const bf16_t *v_cache,
                                       const int *block_tables, const int *ctx_lens, int S, int nq, int nkv, int hd,
                                       int max_blocks, int block_size, float scale, int window, int sinks, int max_ctx,
                                       void *work, size_t work_bytes) {
    const char *who = "attn_decode_window";
    if (S <= 0 || !check_attention(who, out, q, k_cache, v_cache, block_tables, ctx_lens, nq, nkv, hd, max_blocks,
                                   block_size, scale, window, sinks, work))
        return;
    if (!launch_split_rows(RowArgs{out, q, k_cache, v_cache, block_tables, ctx_lens, nullptr, nullptr, S, nq, nkv,
                                   max_blocks, block_size,
                                   (block_size & (block_size - 1)) == 0 ? __builtin_ctz(block_size) : -1,
                                   scale * LLMGEN_LOG2E, window ? std::min(window, NO_WINDOW) : NO_WINDOW,
                                   std::min(sinks, NO_WINDOW)},
                           S, max_ctx, split_work(work, work_bytes)))
        refuse(who, "too many sequences");
}

extern "C" void hip_attn_prefill_window(bf16_t *out, const bf16_t *q, const bf16_t *k_cache, const bf16_t *v_cache,
                                        const int *block_tables, const int *ctx_lens, const int *cu_q,
                                        const int *tile_seq, const int *tile_q0, int n_tiles, int nq, int nkv, int hd,
                                        int max_blocks, int block_size, float scale, int window, int sinks,
                                        int single_rows, void *work, size_t work_bytes) {
    prefill("attn_prefill_window", false, out, q, k_cache, v_cache, block_tables, ctx_lens, cu_q, tile_seq, tile_q0,
            n_tiles, nq, nkv, hd, max_blocks, block_size, scale, window, sinks, single_rows, work, work_bytes);
}

extern "C" void hip_attn_prefill_kv4(bf16_t *out, const bf16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                                     const int *block_tables, const int *ctx_lens, const int *cu_q, const int *tile_seq,
                                     const int *tile_q0, int n_tiles, int nq, int nkv, int hd, int max_blocks,
                                     int block_size, float scale, int window, int sinks, int single_rows, void *work,
                                     size_t work_bytes) {
    prefill("attn_prefill_kv4", true, out, q, k_cache, v_cache, block_tables, ctx_lens, cu_q, tile_seq, tile_q0, n_tiles,
            nq, nkv, hd, max_blocks, block_size, scale, window, sinks, single_rows, work, work_bytes);
}
