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
    int n_tiles, nq, nkv, G, head_groups, max_blocks, block_size, bs_shift;
    float scale_log2;
    int window, sinks;
    bool single;  // segments of one row are computed here (no decode launch for them)
};

// The workgroup's work: unit `bid` of the grid (KV head fastest, then group of NW / 2 heads, then tile from the end of
// the list), key tiles [j0, j1) of it (j1 < 0: to its last).  If part is not null the partial result goes there
// (device-coherent stores, NW * PART_WAVE_FLOATS floats, the layout prefill_merge_store_n reads) instead of rows to out.
template <int NW, int MODE>
__device__ __forceinline__ void window_body(const WindowArgs &a, int bid, unsigned char *lds, int j0, int j1,
                                            float *__restrict__ part) {
    constexpr int LOADS = 16 / NW;  // 4-row DMA instructions per wave per tile, for K and for V each
    WindowLds<NW> &sm = *reinterpret_cast<WindowLds<NW> *>(lds);
    constexpr bool ONE_STAGE = WindowLds<NW>::ONE_STAGE;
    bf16_t *K0 = sm.K0, *V0 = sm.V0, *K1 = ONE_STAGE ? sm.K0 : sm.K1, *V1 = ONE_STAGE ? sm.V0 : sm.V1;

    const int nq = a.nq, nkv = a.nkv, block_size = a.block_size, bs_shift = a.bs_shift;
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
    if (ctx < q_len) {                    // padding sequence: zero rows, no keys
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
    //      swizzles onto it ----
    const int drow = lane >> 4, dchunk = lane & 15;
    auto issue = [&](int it, bf16_t *Kd, bf16_t *Vd) {
        const bf16_t *kc = static_cast<const bf16_t *>(a.kc), *vc = static_cast<const bf16_t *>(a.vc);
        const long blk_stride = (long)nkv * block_size * HD;
        const long head_off = (long)kvh * block_size * HD;
        const int kb0 = tile_key(it);
        const int last = kend - 1 - kb0;
        __amdgpu_buffer_rsrc_t krs, vrs;
        if (MODE == DMA_BLOCK) {  // the whole tile lies in one block: one descriptor pair per tile
            const int phys = bt[__builtin_amdgcn_readfirstlane(kb0 >> bs_shift)];
            const long base = (long)phys * blk_stride + head_off + (long)(kb0 & (block_size - 1)) * HD;
            krs = make_rsrc(kc + base, TILE * 2);
            vrs = make_rsrc(vc + base, TILE * 2);
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
                const int bi = bs_shift >= 0 ? (t0 >> bs_shift) : t0 / block_size;
                const long base = (long)bt[bi] * blk_stride + head_off + (long)(t0 - bi * block_size) * HD;
                const int voff = (src - first) * (HD * 2);
                bufdma16(make_rsrc(kc + base, 4 * HD * 2), voff + kswz, Kd + rbase * HD);
                bufdma16(make_rsrc(vc + base, 4 * HD * 2), voff + vswz, Vd + rbase * HD);
            } else {
                const int t = kb0 + src;
                const int bi = t / block_size;
                const long at = (long)bt[bi] * blk_stride + head_off + (long)(t - bi * block_size) * HD;
                dma16(kc + at + (kswz >> 1), Kd + rbase * HD);
                dma16(vc + at + (vswz >> 1), Vd + rbase * HD);
            }
        }
    };

    // ---- 4-bit pages: a tile is 64 rows x 4 runs of 32 values (16 bytes of codes and a scale byte) of K, then of V;
    //      thread i takes runs i, i + 64 NW, ...  fetch() loads them into registers, commit() converts them into a stage
    constexpr int RUNS = MODE == KV4 ? 8 / NW : 1;
    u32x4_t run_codes[RUNS];
    uint32_t run_scale[RUNS];
    auto fetch = [&](int it) {
        const int kb0 = tile_key(it), last = kend - 1 - kb0;
        const long hb = llmgen_cache::head_bytes(block_size);
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const int c = tid + i * 64 * NW, r = (c & 255) >> 2, run = c & 3;
            const int t = kb0 + seen_row(r, kb0, kt.lo, sinks, last);
            const int bi = bs_shift >= 0 ? t >> bs_shift : t / block_size;
            const int off = t - bi * block_size;
            const uint8_t *p = static_cast<const uint8_t *>(c < 256 ? a.kc : a.vc) + ((long)bt[bi] * nkv + kvh) * hb;
            run_codes[i] = ld16(p + (long)off * llmgen_cache::CODE_BYTES + run * 16);
            run_scale[i] = p[(long)block_size * llmgen_cache::CODE_BYTES + (long)off * llmgen_cache::SCALE_BYTES + run];
        }
    };
    auto commit = [&](bf16_t *Kd, bf16_t *Vd) {
#pragma unroll
        for (int i = 0; i < RUNS; ++i) {
            const int c = tid + i * 64 * NW, r = (c & 255) >> 2, run = c & 3;
            const float sc = llmgen_cache::kv4_scale(run_scale[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                bf16_t *dst = c < 256 ? Kd + k_off(r, run * 4 + j) : Vd + v_off(r, run * 4 + j);
                *reinterpret_cast<u32x4_t *>(dst) = llmgen_cache::kv4_to_bf16(run_codes[i][j], sc);
            }
        }
    };

    f32x16_t o[4];
    float m_run, l_run;
    bool careful = false;  // the second run of a unit that met an infinity or NaN

    // per-lane LDS offsets of the V^T fragment reads (ds_read_b64_tr_b16): 16-lane group g4, lane i = 4j + m;
    // the fragment's k-slots (hh*8 + e) are keys kc16*16 + (e/4)*8 + hh*4 + e%4, so the two reads of a fragment
    // take keys hh*4 + j (+8) and dims db*32 + (g4&1)*16 + 4m .. +3
    int voff[4];
    {
        const int g4 = lane >> 4, i = lane & 15, j = i >> 2, m = i & 3;
        const int key = (g4 >> 1) * 4 + j;
#pragma unroll
        for (int db = 0; db < 4; ++db) {
            const int dim = db * 32 + (g4 & 1) * 16 + 4 * m;
            voff[db] = v_off(key, dim >> 3) + (dim & 7);
        }
    }
    // per-lane LDS offsets of the K fragment reads (row l32, logical chunk 2c + hh); row 32 + l32 has the same
    // swizzle, so its offset is a constant 32 rows further
    int koff[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) koff[c] = k_off(l32, 2 * c + hh);

    // One 64-key tile for this wave: S^T = K Q^T, online softmax (base 2, scale folded into one FMA), O^T += V^T P^T.
    auto tile_step = [&](int kb0, const bf16_t *Ks, const bf16_t *Vs, auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        // offset `off` of this lane's keys (key kb0 + off + hh*4) is hidden from its row when it lies past the row's
        // position (or the row is padding), or before its window and behind the sinks
        const int lim = row_valid ? my_pos - kb0 - hh * 4 : -1;
        const int lim_lo = my_pos - window - kb0 - hh * 4, lim_s = sinks - kb0 - hh * 4;
        auto hidden = [&](int off) { return off > lim || (off <= lim_lo && off >= lim_s); };
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
            const bf16_t *vp = Vs + (i >> 2) * 16 * HD + voff[i & 3];
            const s16x4_t lo = ds_read_tr(vp);           // keys hh*4 + j
            const s16x4_t hi = ds_read_tr(vp + 8 * HD);  // keys 8 + hh*4 + j
            va[i] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        };
#pragma unroll
        for (int i = 0; i < VPF; ++i) vread(i);
        __builtin_amdgcn_sched_barrier(0);
        // lane holds row my_row, keys kb0 + kb*32 + (r/4)*8 + hh*4 + r%4 (raw dot products)
        if (MASK) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (hidden(kb * 32 + (r >> 2) * 8 + (r & 3))) sacc[kb][r] = -INFINITY;
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
        // a row max (they may exceed 1: o / l is unchanged by the common factor).  Only a row sum beyond 2^64 moves the
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
            if (__any(!(lsum <= 0x1p64f))) {
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
        if constexpr (MASK) {
            if (careful) {
                typedef uint16_t u16x8_t __attribute__((ext_vector_type(8)));
                bf16x8_t see[4];  // 1 for this lane's keys that its row sees, laid out as the probabilities are
#pragma unroll
                for (int kc16 = 0; kc16 < 4; ++kc16)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int r = (kc16 & 1) * 8 + e;
                        see[kc16][e] = (__bf16)(hidden((kc16 >> 1) * 32 + (r >> 2) * 8 + (r & 3)) ? 0.f : 1.f);
                    }
#pragma unroll
                for (int db = 0; db < 4; ++db) {
                    // the finite values, and how many visible keys hold +inf, -inf and NaN in each place
                    f32x16_t count[3];
#pragma unroll
                    for (int w = 0; w < 3; ++w)
#pragma unroll
                        for (int r = 0; r < 16; ++r) count[w][r] = 0.f;
#pragma unroll
                    for (int kc16 = 0; kc16 < 4; ++kc16) {
                        vread(kc16 * 4 + db);
                        const u16x8_t v = __builtin_bit_cast(u16x8_t, va[kc16 * 4 + db]);
                        u16x8_t f = v;
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if ((v[e] & 0x7f80u) == 0x7f80u) f[e] = 0;
                        o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, f), pf[kc16], o[db],
                                                                        0, 0, 0);
#pragma unroll
                        for (int w = 0; w < 3; ++w) {
                            u16x8_t is;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const bool hit = w == 0 ? v[e] == 0x7f80u : w == 1 ? v[e] == 0xff80u : (v[e] & 0x7fffu) > 0x7f80u;
                                is[e] = hit ? 0x3f80u : 0;  // 1 or 0
                            }
                            count[w] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, is), see[kc16],
                                                                               count[w], 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        if (count[0][r] > 0.f) o[db][r] += INFINITY;
                        if (count[1][r] > 0.f) o[db][r] -= INFINITY;
                        if (count[2][r] > 0.f) o[db][r] = NAN;
                    }
                }
                return;
            }
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
        // tiles that every row of the wave sees whole take the unmasked path
        if (wave_has_pad || kb0 + BK - 1 > wave_pos_min || (kb0 <= wave_pos_max - window && kb0 + BK > sinks))
            tile_step(kb0, Ks, Vs, std::true_type{});
        else
            tile_step(kb0, Ks, Vs, std::false_type{});
    };

    for (int run = 0;; ++run) {
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[db][r] = 0.f;
        m_run = -INFINITY;
        l_run = 0.f;
        if constexpr (MODE == KV4) {
            fetch(0);
            for (int it = 0; it < n_iter; it += 2) {
                commit(K0, V0);
                __syncthreads();  // the tile is there, and everyone is done with the stage written next
                if (it + 1 < n_iter) fetch(it + 1);
                compute(it, K0, V0);
                if (ONE_STAGE) __syncthreads();
                if (it + 1 >= n_iter) break;
                commit(K1, V1);
                __syncthreads();
                if (it + 2 < n_iter) fetch(it + 2);
                compute(it + 1, K1, V1);
                if (ONE_STAGE) __syncthreads();
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
        if (run == 1) break;
        float z = 0.f;  // stays 0 unless an accumulator of a row of the segment is an infinity or NaN
        if (wave_active && row_valid) {
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) z = __builtin_fmaf(o[db][r], 0.f, z);
        }
        if (!__syncthreads_or(!(z == 0.f))) break;
        careful = true;
    }

    if (part) {  // leave the partial result (the merging workgroup reads it with device-coherent loads)
        if (!wave_active) return;
        float *pw = part + wave * PART_WAVE_FLOATS + lane;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                __hip_atomic_store(pw + (db * 16 + r) * 64, o[db][r], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(pw + 64 * 64, m_run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __hip_atomic_store(pw + 65 * 64, l_run, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        return;
    }
    // ---- normalise and store: lane holds dims db*32 + (r/4)*8 + hh*4 + r%4 of row my_row ----
    if (!wave_active) return;
    const float l_tot = l_run + lane_xor(l_run, 32);
    if (!row_valid) return;
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

}  // namespace llmgen_window
