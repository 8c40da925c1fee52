// window_kernel.h -- the prefill workgroup over a cache with a sliding window and sinks, on bf16 or 4-bit pages (gfx950).
// What it computes and how is described in window.hip; the tile layouts and fragment reads are those of
// prefill_kernel.h.
#pragma once
#include "cache_common.h"
#include "hip_common.h"
#include "prefill_kernel.h"

#include <math.h>

#include <type_traits>

namespace llmgen_window {

using namespace llmgen_prefill;

// How a tile of keys reaches LDS: the DMA modes of bf16 pages, or 4-bit pages of any block size, whose rows pass through
// registers and are converted to bf16 on the way.
constexpr int KV4 = 3;

// The key tiles of a unit whose first row sits at position pos0 and whose last key is kend - 1: sink_tiles tiles from
// key 0 on, then, gap tiles further, those from the tile of lo, the first key that the first row sees through the
// window; n in all.
struct KeyTiles {
    int lo, sink_tiles, gap, n;
};
__device__ __forceinline__ KeyTiles key_tiles(int pos0, int kend, int window, int sinks) {
    KeyTiles k;
    k.lo = max(0, pos0 - window + 1);
    k.sink_tiles = min((sinks + BK - 1) / BK, k.lo / BK);
    k.gap = k.lo / BK - k.sink_tiles;
    k.n = (kend + BK - 1) / BK - k.gap;
    return k;
}
// The row to read for row r of the tile at key kb0: r itself where some row of the unit sees that key (a sink, or lo and
// later, up to row `last`), else a row that is seen -- of r's four if one of them is, so that the four rows of one DMA
// instruction keep one page.
__device__ __forceinline__ int seen_row(int r, int kb0, int lo, int sinks, int last) {
    const int rb = r & ~3, rs = sinks - kb0, rl = lo - kb0;  // rows [rs, rl) are not seen
    int x = r;
    if (r >= rs && r < rl) x = rb < rs ? rs - 1 : rb + 3 >= rl || rl < BK ? rl : rs - 1;
    return min(x, last);
}

// bufdma16 with a wave-uniform byte offset of its own
__device__ __forceinline__ void bufdma16s(__amdgpu_buffer_rsrc_t rs, int voff, int soff, bf16_t *ldst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void *)ldst, 16, voff, soff, 0, 0);
}

// Element offset of (row, 16-byte chunk) in a K or V tile.  Tiles that DMA fills have the layouts of prefill_kernel.h;
// those of 4-bit pages are written by lanes.  There 8 consecutive lanes write the same chunk of 4 runs of rows r and r + 4
// (16 lanes: of r + 8 and r + 12 too), fragment reads of K take one chunk of 8 or 16 neighbouring rows, those of V two
// chunks of 4 rows (four, in 32 lanes): with the run in the low bits of the place and the row added to all of it by XOR,
// each of these covers 8 or 16 places that differ, and so all banks (8192 rows: 541 us without
// conflicts, 547 us with two lanes' writes to a bank).
template <int MODE>
__device__ __forceinline__ int k_place(int row, int chunk) {
    if (MODE != KV4) return k_off(row, chunk);
    return row * HD + ((((chunk & 3) << 2 | chunk >> 2) ^ (row & 15)) << 3);
}
template <int MODE>
__device__ __forceinline__ int v_place(int row, int chunk) {
    return MODE != KV4 ? v_off(row, chunk) : k_place<KV4>(row, chunk);
}

template <int NW>
struct WindowLds {
    // two stages of one 64-key K and V tile; 2-wave workgroups keep one, so that four share a CU
    static constexpr bool ONE_STAGE = NW == 2;
    __attribute__((aligned(16))) bf16_t K0[TILE];
    __attribute__((aligned(16))) bf16_t V0[TILE];
    __attribute__((aligned(16))) bf16_t K1[ONE_STAGE ? 8 : TILE];
    __attribute__((aligned(16))) bf16_t V1[ONE_STAGE ? 8 : TILE];
};

struct WindowArgs {
    bf16_t *out;
    const bf16_t *q;
    const void *kc, *vc;
    const int *block_tables, *ctx_lens, *cu_q, *tile_seq, *tile_q0;
    int n_tiles, nq, nkv, G, head_groups, max_blocks;
    llmgen_cache::PageDiv div;
    float scale_log2;
    int window, sinks;
    bool single;  // segments of one row are computed here (no decode launch for them)
};

// A partial result: for each wave of the workgroup 16 runs of 64 lanes x 4 values of O -- lane hh * 32 + row, run db * 4 +
// rr: dims db * 32 + rr * 8 + hh * 4 on -- then m and l of each lane (PART_WAVE_FLOATS in all).  They pass between
// workgroups while both run, so loads and stores are device-coherent, of 16 bytes a lane (buffer instructions with sc1,
// as the agent-scope atomics have, which there are for 8 bytes at most).
constexpr int SC1 = 16;

// One query row (at element `row` of q and out, position pos) over n tiles from j0 on, by one wave: lane = key for the
// scores, lane = two values of the head for the sums, online softmax in base 2.  Reads only keys that the row sees.  The
// result goes to out, or as row r of a wave's partial result.
template <int MODE>
__device__ __forceinline__ void redo_row(const WindowArgs &a, const int *bt, int kvh, long row, int pos, const KeyTiles &kt,
                                         int j0, int n, float *part, int r) {
    const int lane = threadIdx.x & 63;
    const long hb = MODE == KV4 ? llmgen_cache::head_bytes(a.div.bs) : (long)a.div.bs * HD * 2;
    auto place = [&](int t, int &off) {  // key t's page and head, and its row there
        const int blk = a.div(t);
        off = t - blk * a.div.bs;
        return ((long)bt[blk] * a.nkv + kvh) * hb;
    };
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        const int ti = j0 + i, kb0 = (ti >= kt.sink_tiles ? ti + kt.gap : ti) * BK, t = kb0 + lane;
        const bool vis = t <= pos && (t > pos - a.window || t < a.sinks);
        float s = -INFINITY;
        if (vis) {
            int off;
            const uint8_t *p = static_cast<const uint8_t *>(a.kc) + place(t, off);
            s = 0.f;
#pragma unroll 1
            for (int run = 0; run < 4; ++run) {
                u32x4_t codes;
                float sc = 0.f;
                if (MODE == KV4) {
                    codes = ld16(p + (long)off * llmgen_cache::CODE_BYTES + run * 16);
                    sc = llmgen_cache::kv4_scale(p[(long)a.div.bs * llmgen_cache::CODE_BYTES +
                                                   (long)off * llmgen_cache::SCALE_BYTES + run]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float kf[8], qf[8];
                    unpack_bf16x8(MODE == KV4 ? llmgen_cache::kv4_to_bf16(codes[c], sc)
                                              : ld16(p + (long)off * (HD * 2) + run * 64 + c * 16), kf);
                    unpack_bf16x8(ld16(a.q + row + run * 32 + c * 8), qf);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s = __builtin_fmaf(kf[e], qf[e], s);
                }
            }
            s *= a.scale_log2;
        }
        float mx = s;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, lane_xor(mx, d));
        const float m_new = fmaxf(m, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float corr = fast_exp2(m - m_use), p = fast_exp2(s - m_use);
        float sum = p;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) sum += lane_xor(sum, d);
        l = l * corr + sum;
        o0 *= corr;
        o1 *= corr;
        m = m_new;
        for (uint64_t left = __ballot(vis); left; left &= left - 1) {
            const int j = __builtin_ctzll(left);
            const float pj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j));
            int off;
            const uint8_t *v = static_cast<const uint8_t *>(a.vc) + place(kb0 + j, off);
            uint32_t w;
            if (MODE == KV4) {
                const uint32_t code = v[(long)off * llmgen_cache::CODE_BYTES + lane];
                w = llmgen_cache::kv4_to_bf16(code, llmgen_cache::kv4_scale(
                    v[(long)a.div.bs * llmgen_cache::CODE_BYTES + (long)off * llmgen_cache::SCALE_BYTES + lane / 16]))[0];
            } else {
                w = *reinterpret_cast<const uint32_t *>(v + (long)off * (HD * 2) + lane * 4);
            }
            o0 = __builtin_fmaf(pj, bf16lo_to_f32(w), o0);
            o1 = __builtin_fmaf(pj, bf16hi_to_f32(w), o1);
        }
    }
    if (!part) {
        *reinterpret_cast<uint32_t *>(a.out + row + lane * 2) = pack_bf16x2(o0 / l, o1 / l);
        return;
    }
    // values d, d + 1 of row r lie in run (d / 32) * 4 + d / 8 % 4 of lane (d / 4 % 2) * 32 + r, from its d % 4 on
    const int d = lane * 2;
    float *at = part + ((d >> 5) * 4 + (d >> 3 & 3)) * 256 + ((d >> 2 & 1) * 32 + r) * 4 + (d & 3);
    __hip_atomic_store(at, o0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(at + 1, o1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (lane < 2) {  // the merge adds the halves' l
        __hip_atomic_store(part + 64 * 64 + lane * 32 + r, m, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(part + 65 * 64 + lane * 32 + r, lane ? 0.f : l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

// The workgroup's work: unit `bid` of the grid (KV head fastest, then group of NW / 2 heads, then tile from the end of
// the list), key tiles [j0, j1) of it (j1 < 0: to its last).  If part is not null the partial result goes there
// (NW * PART_WAVE_FLOATS floats) instead of rows to out.
//
// Masking a score does not stop an infinity or NaN in V, as 0 times it is NaN.  Rows whose accumulators end up with one
// (and whose scores have none: then the result is NaN) are therefore computed again by redo_row, which multiplies only
// values that the row sees.
template <int NW, int MODE>
__device__ __forceinline__ void window_body(const WindowArgs &a, int bid, unsigned char *lds, int j0, int j1,
                                            float *__restrict__ part) {
    constexpr int LOADS = 16 / NW;  // 4-row DMA instructions per wave per tile, for K and for V each
    WindowLds<NW> &sm = *reinterpret_cast<WindowLds<NW> *>(lds);
    constexpr bool ONE_STAGE = WindowLds<NW>::ONE_STAGE;
    bf16_t *K0 = sm.K0, *V0 = sm.V0, *K1 = ONE_STAGE ? sm.K0 : sm.K1, *V1 = ONE_STAGE ? sm.V0 : sm.V1;

    const int nq = a.nq, nkv = a.nkv, block_size = a.div.bs;
    const int window = a.window, sinks = a.sinks;
    const float scale_log2 = a.scale_log2;
    const int kvh = bid % nkv;
    const int rest = bid / nkv;
    const int hg = rest % a.head_groups;
    const int tile = a.n_tiles - 1 - rest / a.head_groups;
    const int s = a.tile_seq[tile], q0 = a.tile_q0[tile];
    const int q_beg = a.cu_q[s], q_len = a.cu_q[s + 1] - q_beg;
    const int ctx = (int)min((long)a.ctx_lens[s], (long)a.max_blocks * block_size);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int head = kvh * a.G + hg * (NW / 2) + (wave >> 1);
    const int r0 = q0 + (wave & 1) * 32;  // first query row (within the segment) of this wave
    const int l32 = lane & 31, hh = lane >> 5;

    if (q_len == 1 && !a.single) return;  // streamed by the decode launch
    if (ctx < q_len) {                          // padding sequence: zero rows, no keys
        const int row = r0 + l32;
        if (row < q_len) {
            bf16_t *o = a.out + ((long)(q_beg + row) * nq + head) * HD + hh * 64;
            for (int d = 0; d < 64; d += 8) *reinterpret_cast<u32x4_t *>(o + d) = u32x4_t{0, 0, 0, 0};
        }
        return;
    }

    const int *bt = a.block_tables + (long)s * a.max_blocks;
    const int base_pos = ctx - q_len;                  // position of segment row 0
    const int kend = base_pos + min(q0 + BQ, q_len);   // keys needed by the whole tile
    const KeyTiles kt = key_tiles(base_pos + q0, kend, window, sinks);
    const int n_iter = (j1 >= 0 ? min(j1, kt.n) : kt.n) - j0;
    auto tile_key = [&](int it) {  // first key of iteration it's tile
        const int ti = j0 + it;
        return (ti >= kt.sink_tiles ? ti + kt.gap : ti) * BK;
    };

    // ---- Q fragments (B operand): lane holds row r0+l32, dims c*16 + hh*8 .. +8 ----
    const int my_row = r0 + l32;
    const bool row_valid = my_row < q_len;
    const int my_pos = base_pos + my_row;
    bf16x8_t qf[8];
    {
        const int rq = min(my_row, q_len - 1);
        const bf16_t *qp = a.q + ((long)(q_beg + rq) * nq + head) * HD + hh * 8;
#pragma unroll
        for (int c = 0; c < 8; ++c) qf[c] = __builtin_bit_cast(bf16x8_t, ld16(qp + c * 16));
    }
    const bool wave_active = r0 < q_len;
    const int wave_pos_min = base_pos + r0;
    const int wave_pos_max = base_pos + min(r0 + 31, q_len - 1);
    const bool wave_has_pad = r0 + 31 >= q_len;

    // ---- bf16 pages: DMA of the K/V tile of iteration `it` into (Kd, Vd): wave instruction i covers rows
    //      4*(wave + NW*i) .. +3; lane writes row + lane/16, physical chunk lane%16, so it reads the logical chunk that
    //      swizzles onto it.
    //
    // Pages are looked up ahead of use, by vector loads: a scalar load in flight makes every wait for an LDS read a wait
    // for all of them and for itself (both count on lgkmcnt), which cost 20 % of the time.  Where a wave needs one page
    // a tile (BLOCK) or a DMA instruction (ROW4), lane l looks up entry l % LOOKS of tile l / LOOKS of the next PER
    // tiles, PER tiles ahead, and the pages are read out as scalars; else each lane looks its own rows' pages up, a
    // tile ahead. ----
    const int drow = lane >> 4, dchunk = lane & 15;
    // 4-bit pages: rows of a tile whose runs a thread takes (4 consecutive threads share a row, 16 take rows 4 apart)
    constexpr int RUN_ROWS = NW == 2 ? 2 : 1;
    const int run4 = tid >> 2, my_run_row = (run4 & ~15) | (run4 & 3) << 2 | (run4 >> 2 & 3);
    const long hb = llmgen_cache::head_bytes(block_size);
    constexpr bool BY_LANE = MODE == DMA_BLOCK || MODE == DMA_ROW4;
    constexpr int LOOKS = MODE == KV4 ? RUN_ROWS : MODE == DMA_BLOCK ? 1 : LOADS, PER = BY_LANE ? 64 / LOOKS : 1;
    int blk[BY_LANE ? 2 : LOOKS];  // BY_LANE: this lane's page of the current tiles and of the next ones
    auto lookup = [&](int it) {
        if (it >= n_iter) return;
        if constexpr (BY_LANE) {
            const int at = min(it + lane / LOOKS, n_iter - 1);
            const int kb0 = tile_key(at), last = kend - 1 - kb0;
            const int r = MODE == DMA_BLOCK ? 0 : seen_row(4 * (wave + NW * (lane % LOOKS)), kb0, kt.lo, sinks, last);
            blk[1] = bt[a.div(kb0 + r)];
        } else {
            const int kb0 = tile_key(it), last = kend - 1 - kb0;
#pragma unroll
            for (int i = 0; i < LOOKS; ++i) {
                const int r = MODE == KV4 ? my_run_row + 32 * i : 4 * (wave + NW * i) + drow;
                blk[i] = bt[a.div(kb0 + seen_row(r, kb0, kt.lo, sinks, last))];
            }
        }
    };
    auto page = [&](int it, int i) {
        return BY_LANE ? __builtin_amdgcn_readlane(blk[0], it % PER * LOOKS + i) : blk[i % LOOKS];
    };
    constexpr int KSWZ = NW == 2 ? 2 : 1;
    int k_lane[KSWZ], v_lane;
    {
        const int first = MODE == DMA_BLOCK ? 4 * wave + drow : drow;  // from the descriptor's row
#pragma unroll
        for (int i = 0; i < KSWZ; ++i)
            k_lane[i] = first * (HD * 2) + ((dchunk ^ ((4 * (wave + NW * i) + drow) & 15)) << 4);
        v_lane = first * (HD * 2) + ((dchunk ^ ((drow << 2) & 15)) << 4);
    }
    auto issue = [&](int it, bf16_t *Kd, bf16_t *Vd) {
        const bf16_t *kc = static_cast<const bf16_t *>(a.kc), *vc = static_cast<const bf16_t *>(a.vc);
        const long blk_stride = (long)nkv * block_size * HD;
        const long head_off = (long)kvh * block_size * HD;
        const int kb0 = tile_key(it);
        const int last = kend - 1 - kb0;
        if (BY_LANE && it % PER == 0) {
            blk[0] = blk[1];
            lookup(it + PER);
        }
        __amdgpu_buffer_rsrc_t krs, vrs;
        if (MODE == DMA_BLOCK) {  // the whole tile lies in one block: one descriptor pair per tile
            const long base = (long)page(it, 0) * blk_stride + head_off + (long)(kb0 & (block_size - 1)) * HD;
            krs = make_rsrc(kc + base, TILE * 2);
            vrs = make_rsrc(vc + base, TILE * 2);
        }
        if (BY_LANE && (kb0 >= kt.lo || kb0 + BK <= sinks) && last >= BK - 1) {
            // every row of the tile is read: the lanes' offsets are the same in each such tile.  They repeat from one
            // instruction to the next (every second one where 4 NW rows are half a swizzle period)
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int rbase = 4 * (wave + NW * i), soff = NW * 4 * (HD * 2) * i;
                if (MODE == DMA_BLOCK) {
                    bufdma16s(krs, k_lane[i % KSWZ], soff, Kd + rbase * HD);
                    bufdma16s(vrs, v_lane, soff, Vd + rbase * HD);
                } else {
                    const int t0 = __builtin_amdgcn_readfirstlane(kb0 + rbase);
                    const long base =
                        (long)page(it, i) * blk_stride + head_off + (long)(t0 - a.div(t0) * block_size) * HD;
                    bufdma16(make_rsrc(kc + base, 4 * HD * 2), k_lane[i % KSWZ], Kd + rbase * HD);
                    bufdma16(make_rsrc(vc + base, 4 * HD * 2), v_lane, Vd + rbase * HD);
                }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int rbase = 4 * (wave + NW * i);
            const int r = rbase + drow;
            const int src = seen_row(r, kb0, kt.lo, sinks, last);
            const int kswz = (dchunk ^ (r & 15)) << 4, vswz = (dchunk ^ ((r << 2) & 15)) << 4;  // bytes
            if (MODE == DMA_BLOCK) {
                bufdma16(krs, src * (HD * 2) + kswz, Kd + rbase * HD);
                bufdma16(vrs, src * (HD * 2) + vswz, Vd + rbase * HD);
            } else if (MODE == DMA_ROW4) {
                const int first = seen_row(rbase, kb0, kt.lo, sinks, last);
                const int t0 = __builtin_amdgcn_readfirstlane(kb0 + first);
                const long base =
                    (long)page(it, i) * blk_stride + head_off + (long)(t0 - a.div(t0) * block_size) * HD;
                const int voff = (src - first) * (HD * 2);
                bufdma16(make_rsrc(kc + base, 4 * HD * 2), voff + kswz, Kd + rbase * HD);
                bufdma16(make_rsrc(vc + base, 4 * HD * 2), voff + vswz, Vd + rbase * HD);
            } else {
                const int t = kb0 + src;
                const long at = (long)page(it, i) * blk_stride + head_off + (long)(t - a.div(t) * block_size) * HD;
                dma16(kc + at + (kswz >> 1), Kd + rbase * HD);
                dma16(vc + at + (vswz >> 1), Vd + rbase * HD);
            }
        }
        if (!BY_LANE) lookup(it + 1);
    };

    // ---- 4-bit pages: a tile is 64 rows x 4 runs of 32 values (16 bytes of codes and a scale byte) of K and of V.  A
    //      thread takes run tid % 4 of row my_run_row (and of the row 32 further with 128 threads), of both K and V.
    //      fetch() loads runs into registers, commit() converts them into a stage
    static_assert(MODE != KV4 || NW <= 4, "256 threads take a tile's runs");
    u32x4_t run_codes[RUN_ROWS][2];
    uint32_t run_scale[RUN_ROWS][2];
    auto fetch = [&](int it) {
        const int kb0 = tile_key(it), last = kend - 1 - kb0, run = tid & 3;
        const bool all = (kb0 >= kt.lo || kb0 + BK <= sinks) && last >= BK - 1;  // every row of the tile is read
#pragma unroll
        for (int i = 0; i < (MODE == KV4 ? RUN_ROWS : 0); ++i) {
            const int r = my_run_row + 32 * i;
            const int t = kb0 + (all ? r : seen_row(r, kb0, kt.lo, sinks, last));
            const int off = t - a.div(t) * block_size;
            const long at = ((long)blk[i] * nkv + kvh) * hb;
            const int codes = off * llmgen_cache::CODE_BYTES + run * 16;
            const int scale = block_size * llmgen_cache::CODE_BYTES + off * llmgen_cache::SCALE_BYTES + run;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint8_t *p = static_cast<const uint8_t *>(j ? a.vc : a.kc) + at;
                run_codes[i][j] = ld16(p + codes);
                run_scale[i][j] = p[scale];
            }
        }
        lookup(it + 1);
    };
    auto commit = [&](bf16_t *Kd, bf16_t *Vd) {
#pragma unroll
        for (int i = 0; i < RUN_ROWS; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                bf16_t *dst = j ? Vd : Kd;
                const float sc = llmgen_cache::kv4_scale(run_scale[i][j]);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    *reinterpret_cast<u32x4_t *>(dst + k_place<KV4>(my_run_row + 32 * i, (tid & 3) * 4 + c)) =
                        llmgen_cache::kv4_to_bf16(run_codes[i][j][c], sc);
            }
    };

    f32x16_t o[4];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;

    // per-lane LDS offsets of the V^T fragment reads (ds_read_b64_tr_b16): 16-lane group g4, lane i = 4j + m;
    // the fragment's k-slots (hh*8 + e) are keys kc16*16 + (e/4)*8 + hh*4 + e%4, so the two reads of a fragment
    // take keys hh*4 + j (+8) and dims db*32 + (g4&1)*16 + 4m .. +3
    int voff[4], vhi[4];  // of keys j, and of keys 8 + j
    {
        const int g4 = lane >> 4, i = lane & 15, j = i >> 2, m = i & 3;
        const int key = (g4 >> 1) * 4 + j;
#pragma unroll
        for (int db = 0; db < 4; ++db) {
            const int dim = db * 32 + (g4 & 1) * 16 + 4 * m;
            voff[db] = v_place<MODE>(key, dim >> 3) + (dim & 7);
            vhi[db] = v_place<MODE>(key + 8, dim >> 3) + (dim & 7);
        }
    }
    // per-lane LDS offsets of the K fragment reads (row l32, logical chunk 2c + hh); row 32 + l32 has the same
    // swizzle, so its offset is a constant 32 rows further
    int koff[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) koff[c] = k_place<MODE>(l32, 2 * c + hh);

    // One 64-key tile for this wave: S^T = K Q^T, online softmax (base 2, scale folded into one FMA), O^T += V^T P^T.
    auto tile_step = [&](int kb0, const bf16_t *Ks, const bf16_t *Vs, bool masked) {
        f32x16_t sacc[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) sacc[kb][r] = 0.f;
        bf16x8_t ka[8], kb[8];  // K fragments of keys 0-31 and 32-63, read KPF steps ahead
#pragma unroll
        for (int c = 0; c < KPF; ++c) {
            ka[c] = *reinterpret_cast<const bf16x8_t *>(Ks + koff[c]);
            kb[c] = *reinterpret_cast<const bf16x8_t *>(Ks + koff[c] + 32 * HD);
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {  // two independent accumulation chains interleaved
            if (c + KPF < 8) {
                ka[c + KPF] = *reinterpret_cast<const bf16x8_t *>(Ks + koff[c + KPF]);
                kb[c + KPF] = *reinterpret_cast<const bf16x8_t *>(Ks + koff[c + KPF] + 32 * HD);
            }
            sacc[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ka[c], qf[c], sacc[0], 0, 0, 0);
            sacc[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kb[c], qf[c], sacc[1], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);  // keep the read-ahead order
        }
        // V^T fragment i = kc16 * 4 + db: keys kc16*16 + hh*4 + j (+8), dims db*32 + ...; the first VPF do not
        // depend on P and are read before the softmax
        bf16x8_t va[16];
        auto vread = [&](int i) {
            const bf16_t *vp = Vs + (i >> 2) * 16 * HD;
            const s16x4_t lo = ds_read_tr(vp + voff[i & 3]);  // keys hh*4 + j
            const s16x4_t hi = ds_read_tr(vp + vhi[i & 3]);   // keys 8 + hh*4 + j
            va[i] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
#pragma unroll
        for (int i = 0; i < VPF; ++i) vread(i);
        __builtin_amdgcn_sched_barrier(0);
        // lane holds row my_row, keys kb0 + kb*32 + (r/4)*8 + hh*4 + r%4 (raw dot products)
        if (masked) {
            // Key kb0 + off + hh*4 is hidden from the row when it lies past its position (or the row is padding), or
            // before its window and behind the sinks: one bit an offset, then two instructions a score (the bit spread
            // over a word, and a bitwise select of -inf)
            auto above = [](int x) -> uint64_t {  // bits of the offsets > x
                return x < 0 ? ~0ull : x >= 63 ? 0ull : ~0ull << (x + 1);
            };
            const int at = kb0 + hh * 4;
            const uint64_t hid =
                above(row_valid ? my_pos - at : -1) | (~above(my_pos - window - at) & above(sinks - at - 1));
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const uint32_t bits = (uint32_t)(hid >> (32 * kb));
                    const uint32_t m = (uint32_t)((int)(bits << (31 - ((r >> 2) * 8 + (r & 3)))) >> 31);
                    const float x = sacc[kb][r];
                    sacc[kb][r] = __builtin_bit_cast(float, (m & 0xff800000u) | (~m & __builtin_bit_cast(uint32_t, x)));
                }
        }
        auto row_max = [&]() {
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[kb][r]);
            return fmaxf(mx, lane_xor(mx, 32)) * scale_log2;  // scale > 0 commutes with max
        };
        float lsum;
        bf16x8_t pf[4];  // B fragments for the four 16-key steps of P V
        auto probs = [&](float m_use) {
            lsum = 0.f;
#pragma unroll
            for (int kc16 = 0; kc16 < 4; ++kc16) {
                const int kb = kc16 >> 1, half = kc16 & 1;
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = fast_exp2(__builtin_fmaf(sacc[kb][half * 8 + e], scale_log2, -m_use));
                    lsum += p[e];
                }
                u32x4_t w;
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(p[2 * e], p[2 * e + 1]);
                pf[kc16] = __builtin_bit_cast(bf16x8_t, w);
            }
        };
        // Once every row of the wave has a finite reference m_run, the tile's probabilities are taken against it without
        // a row max (they may exceed 1: o / l is unchanged by the common factor).  Only a row sum beyond 2^16 moves the
        // reference, recomputing the tile against the new row max.
        bool grow = false;
        float m_new = m_run, corr = 1.f;
        if (!__all(m_run > -INFINITY)) {
            const float mx = row_max();
            grow = mx > m_run + RESCALE_LOG2;
            m_new = grow ? mx : m_run;
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            corr = grow ? fast_exp2(m_run - m_use) : 1.f;
            probs(m_use);
        } else {
            probs(m_run);
            if (__any(!(lsum <= 0x1p16f))) {
                const float mx = row_max();
                grow = mx > m_run;
                m_new = grow ? mx : m_run;
                corr = grow ? fast_exp2(m_run - m_new) : 1.f;
                probs(m_new);
            }
        }
        l_run = l_run * corr + lsum;
        m_run = m_new;
        if (__any(grow)) {  // corr == 1 in rows that did not move
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] *= corr;
        }
        // ---- O^T[dim][row] += V^T P^T: four independent accumulators per 16-key step ----
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (i + VPF < 16) vread(i + VPF);
            o[i & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(va[i], pf[i >> 2], o[i & 3], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto compute = [&](int it, const bf16_t *Ks, const bf16_t *Vs) {
        const int kb0 = tile_key(it);
        if (!wave_active || kb0 > wave_pos_max) return;
        if (kb0 + BK - 1 <= wave_pos_min - window && kb0 >= sinks) return;  // before every row's window
        // One copy of the tile's code for masked and unmasked tiles (a branch around the masks): with two, the compiler
        // keeps O in other registers in each and moves it between them, 60 instructions a tile.
        tile_step(kb0, Ks, Vs, wave_has_pad || kb0 + BK - 1 > wave_pos_min ||
                                   (kb0 <= wave_pos_max - window && kb0 + BK > sinks));
    };

    lookup(0);
    if constexpr (MODE == KV4) {
        // The runs of tile it + 1 were fetched a tile ago; they are converted into the other stage ahead of the products
        // of tile it, beside those of the CU's other workgroup
        auto turn = [&](int it, const bf16_t *Ks, const bf16_t *Vs, bf16_t *Kn, bf16_t *Vn) {
            if (it + 1 < n_iter) commit(Kn, Vn);
            if (it + 2 < n_iter) fetch(it + 2);
            compute(it, Ks, Vs);
            __syncthreads();
        };
        fetch(0);
        commit(K0, V0);
        if (!ONE_STAGE && n_iter > 1) fetch(1);
        __syncthreads();
        if constexpr (ONE_STAGE) {
            for (int it = 0; it < n_iter; ++it) {
                if (it + 1 < n_iter) fetch(it + 1);
                compute(it, K0, V0);
                __syncthreads();  // every wave is done reading the tile
                if (it + 1 < n_iter) commit(K0, V0);
                __syncthreads();
            }
        } else {
            for (int it = 0; it < n_iter; it += 2) {
                turn(it, K0, V0, K1, V1);
                if (it + 1 >= n_iter) break;
                turn(it + 1, K1, V1, K0, V0);
            }
        }
    } else if constexpr (ONE_STAGE) {
        for (int it = 0; it < n_iter; ++it) {
            issue(it, K0, V0);
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();  // the tile has landed for every wave
            compute(it, K0, V0);
            __syncthreads();  // every wave is done reading it
        }
    } else {
        // two LDS stages; the loop is unrolled twice so every DMA targets a fixed buffer (the compiler can then see
        // that the reads of one stage never wait for the DMA into the other)
        issue(0, K0, V0);
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        for (int it = 0; it < n_iter; it += 2) {
            if (it + 1 < n_iter) issue(it + 1, K1, V1);
            compute(it, K0, V0);
            __builtin_amdgcn_s_waitcnt(0);  // this wave's DMA into stage 1 has landed
            __syncthreads();                // ... and everyone's; everyone is done reading stage 0
            if (it + 1 >= n_iter) break;
            if (it + 2 < n_iter) issue(it + 2, K0, V0);
            compute(it + 1, K1, V1);
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
        }
    }
    if (!wave_active) return;
    const float l_tot = l_run + lane_xor(l_run, 32);
    uint64_t again;  // rows to compute again (bits 0-31)
    {
        float z = 0.f;  // stays 0 unless an accumulator is an infinity or NaN
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) z = __builtin_fmaf(o[db][r], 0.f, z);
        again = __ballot(row_valid && !(z == 0.f) && l_tot == l_tot);
        again = (again | again >> 32) & 0xffffffffu;
    }
    const bool mine = row_valid && !(again >> l32 & 1);

    if (part) {  // leave the partial result (the merging workgroup reads it with device-coherent loads)
        if (mine || !row_valid) {
            const __amdgpu_buffer_rsrc_t ps =
                make_rsrc(reinterpret_cast<const bf16_t *>(part), NW * PART_WAVE_FLOATS * (int)sizeof(float));
            const int at = wave * PART_WAVE_FLOATS * (int)sizeof(float) + lane * 16;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const f32x4_t x = {o[i >> 2][(i & 3) * 4], o[i >> 2][(i & 3) * 4 + 1], o[i >> 2][(i & 3) * 4 + 2],
                                   o[i >> 2][(i & 3) * 4 + 3]};
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), ps, at, i * 1024, SC1);
            }
            float *pw = part + wave * PART_WAVE_FLOATS + lane;
            __hip_atomic_store(pw + 64 * 64, m_run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_store(pw + 65 * 64, l_run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    } else if (mine) {  // normalise and store: lane holds dims db*32 + (r/4)*8 + hh*4 + r%4 of row my_row
        const float inv = 1.f / l_tot;
        bf16_t *orow = a.out + ((long)(q_beg + my_row) * nq + head) * HD + hh * 4;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int rr = 0; rr < 4; ++rr) {
                u32x2_t w;
                w[0] = pack_bf16x2(o[db][rr * 4 + 0] * inv, o[db][rr * 4 + 1] * inv);
                w[1] = pack_bf16x2(o[db][rr * 4 + 2] * inv, o[db][rr * 4 + 3] * inv);
                *reinterpret_cast<u32x2_t *>(orow + db * 32 + rr * 8) = w;
            }
    }
    for (; again; again &= again - 1) {
        const int r = __builtin_ctzll(again);
        redo_row<MODE>(a, bt, kvh, ((long)(q_beg + r0 + r) * nq + head) * HD, base_pos + r0 + r, kt, j0, n_iter,
                       part ? part + wave * PART_WAVE_FLOATS : nullptr, r);
    }
}

// The sum of np partial results (at most FAN), `stride` bytes apart from base on, of unit `unit`, taken in order: the
// unit's rows, or (`to` not null) a partial result again.  The loads of one run while the one before it is added.
constexpr int FAN = 8;
template <int NW>
__device__ __forceinline__ void merge_parts(const WindowArgs &a, int unit, const float *base, int stride, int np,
                                            float *to) {
    const int kvh = unit % a.nkv, rest = unit / a.nkv, hg = rest % a.head_groups;
    const int tile = a.n_tiles - 1 - rest / a.head_groups;
    const int s = a.tile_seq[tile], q0 = a.tile_q0[tile];
    const int q_beg = a.cu_q[s], q_len = a.cu_q[s + 1] - q_beg;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int head = kvh * a.G + hg * (NW / 2) + (wave >> 1);
    const int r0 = q0 + (wave & 1) * 32, my_row = r0 + (lane & 31), hh = lane >> 5;
    if (r0 >= q_len) return;  // an inactive wave left no partial
    constexpr int PIECE = NW * PART_WAVE_FLOATS * (int)sizeof(float);  // bytes
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(reinterpret_cast<const bf16_t *>(base), (np - 1) * stride + PIECE);
    const int at = wave * PART_WAVE_FLOATS * (int)sizeof(float);
    f32x4_t x0[16], x1[16], o[16];
    auto load = [&](int p, f32x4_t (&x)[16]) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[i] = __builtin_bit_cast(
                f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, at + lane * 16, p * stride + i * 1024, SC1));
    };
    load(0, x0);
    float w[FAN], lv[FAN];
#pragma unroll
    for (int p = 0; p < FAN; ++p) {
        const int pp = min(p, np - 1);  // no branch: pieces past np reread the last one and are not used
        const uint32_t m = __builtin_amdgcn_raw_buffer_load_b32(rs, at + lane * 4, pp * stride + 64 * 256, SC1);
        const uint32_t l = __builtin_amdgcn_raw_buffer_load_b32(rs, at + lane * 4, pp * stride + 65 * 256, SC1);
        w[p] = __builtin_bit_cast(float, m);
        lv[p] = __builtin_bit_cast(float, l);
    }
    float M = -INFINITY, l = 0.f;
#pragma unroll
    for (int p = 0; p < FAN; ++p) M = fmaxf(M, w[p]);
    const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int p = 0; p < FAN; ++p) {
        w[p] = p < np ? fast_exp2(w[p] - Mu) : 0.f;
        if (p < np) l += lv[p] * w[p];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto add = [&](int p, const f32x4_t (&x)[16]) {
        float c = 0.f;
#pragma unroll
        for (int i = 0; i < FAN; ++i) c = i == p ? w[i] : c;
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] += x[i] * c;
    };
    for (int p = 0; p < np; p += 2) {
        if (p + 1 < np) load(p + 1, x1);
        add(p, x0);
        if (p + 1 >= np) break;
        if (p + 2 < np) load(p + 2, x0);
        add(p + 1, x1);
    }
    if (to) {
        const __amdgpu_buffer_rsrc_t ps = make_rsrc(reinterpret_cast<const bf16_t *>(to), PIECE);
#pragma unroll
        for (int i = 0; i < 16; ++i)
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, o[i]), ps, at + lane * 16, i * 1024, SC1);
        float *pw = to + wave * PART_WAVE_FLOATS + lane;
        __hip_atomic_store(pw + 64 * 64, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(pw + 65 * 64, l, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return;
    }
    const float l_tot = l + lane_xor(l, 32);
    if (my_row >= q_len) return;
    const float inv = 1.f / l_tot;
    bf16_t *orow = a.out + ((long)(q_beg + my_row) * a.nq + head) * HD + hh * 4;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const f32x4_t y = o[i] * inv;
        *reinterpret_cast<u32x2_t *>(orow + i * 8) = u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    }
}

}  // namespace llmgen_window
