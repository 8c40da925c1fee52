// kv4.hip -- the paged KV cache held in 4 bits: writing rows into it, reading them back, and split-K decode over it
// (contracts in include/llmgen_cache.h; the causal prefill over 4-bit pages is in window.hip).
//
// Mathematics: a run of 32 values x shares a power of two 2^e, and value x is held as the e2m1 grid value nearest to
// x / 2^e.  Dequantisation is exact in bf16 (two bits of mantissa and a power of two), so attention over the pages is
// attention over bf16 rows that are read at 68 bytes each instead of 256.
#include "cache_common.h"

#include <algorithm>

namespace {

using namespace llmgen_cache;

// ------------------------------------------------------------------------------------------------------------
// Writing and reading back
// ------------------------------------------------------------------------------------------------------------
// HBM-bound copies with a conversion: 16 lanes take a row, 8 values (16 bytes of bf16, 4 bytes of codes) each, so a wave
// moves 1 KB of bf16 in one access; the largest magnitude of a run of 32 is an integer maximum over the 4 lanes that
// hold it (two DPP steps), and the conversion itself is the hardware's, two values an instruction.  Threads of large
// calls take U = 4 rows, all loads issued before any conversion (16384 tokens x 8 heads,
// 85 MB each: written in 20 us, read back in 15.5 us; with one row a thread 25 and 18 us).
constexpr int ROW_LANES = 16, QUANT_THREADS = 256, ROWS_PER_PASS = QUANT_THREADS / ROW_LANES;

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xF, 0xF, false);
}

// Row r of the call: K's rows (token, kv head), then V's.
struct RowsArgs {
    const int *slots;
    int rows, nkv;
    PageDiv per_token, per_page;  // division by nkv, and by the block size
    long hb;
};
struct RowPlace {
    bool in, live, is_v;  // a row of the call; one with a slot; of V
    int row;              // within K or V
    long codes, scales;  // byte offsets in the pool
};
__device__ __forceinline__ RowPlace row_place(const RowsArgs &a, int r) {
    RowPlace p;
    p.is_v = r >= a.rows;
    p.row = p.is_v ? r - a.rows : r;
    p.in = r < 2 * a.rows;
    const int t = a.per_token(p.row), h = p.row - t * a.nkv;
    const int slot = p.in ? a.slots[t] : -1;
    p.live = slot >= 0;
    const int blk = a.per_page(slot), off = slot - blk * a.per_page.bs;
    const long base = ((long)blk * a.nkv + h) * a.hb;
    p.codes = base + (long)off * CODE_BYTES;
    p.scales = base + (long)a.per_page.bs * CODE_BYTES + (long)off * SCALE_BYTES;
    return p;
}

template <int U>
__global__ void __launch_bounds__(QUANT_THREADS) store_kv4_kernel(const bf16_t *__restrict__ k,
                                                                  const bf16_t *__restrict__ v, uint8_t *__restrict__ kc,
                                                                  uint8_t *__restrict__ vc, const RowsArgs a) {
    const int c = threadIdx.x % ROW_LANES;
    RowPlace p[U];
    u32x4_t x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        p[u] = row_place(a, ((int)blockIdx.x * U + u) * ROWS_PER_PASS + (int)(threadIdx.x / ROW_LANES));
        // not held up by the slot; read once
        if (p[u].in)
            x[u] = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4_t *>((p[u].is_v ? v : k) + (long)p[u].row * HD + c * 8));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (!p[u].live) continue;  // a row's lanes leave together, so the quads below are full
        uint32_t top = kv4_top(x[u]);
        top = max(top, dpp_u<0xB1>(top));
        top = max(top, dpp_u<0x4E>(top));
        const int byte = kv4_scale_byte(top);
        const uint32_t w = kv4_codes(x[u], byte);
        // the row's four scale bytes in one word: rotations by 4 and 8 lanes of the 16
        uint32_t scales = (uint32_t)byte << (c >> 2) * 8;
        scales |= dpp_u<0x124>(scales);
        scales |= dpp_u<0x128>(scales);
        uint8_t *pool = p[u].is_v ? vc : kc;
        *reinterpret_cast<uint32_t *>(pool + p[u].codes + c * 4) = w;
        if (c == 0) *reinterpret_cast<uint32_t *>(pool + p[u].scales) = scales;
    }
}

template <int U>
__global__ void __launch_bounds__(QUANT_THREADS) load_kv4_kernel(bf16_t *__restrict__ k, bf16_t *__restrict__ v,
                                                                 const uint8_t *__restrict__ kc,
                                                                 const uint8_t *__restrict__ vc, const RowsArgs a) {
    const int c = threadIdx.x % ROW_LANES;
    RowPlace p[U];
    uint32_t w[U], s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        p[u] = row_place(a, ((int)blockIdx.x * U + u) * ROWS_PER_PASS + (int)(threadIdx.x / ROW_LANES));
        if (!p[u].live) continue;
        const uint8_t *pool = p[u].is_v ? vc : kc;
        w[u] = *reinterpret_cast<const uint32_t *>(pool + p[u].codes + c * 4);
        s[u] = pool[p[u].scales + (c >> 2)];
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (p[u].live)
            *reinterpret_cast<u32x4_t *>((p[u].is_v ? v : k) + (long)p[u].row * HD + c * 8) =
                kv4_to_bf16(w[u], kv4_scale(s[u]));
}

bool check_rows(const char *who, const void *k, const void *v, const void *slots, const void *kc, const void *vc, int T,
                int nkv, int hd, int block_size) {
    if (!k || !v || !slots || !kc || !vc) return refuse(who, "a tensor is missing");
    if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)kc | (uintptr_t)vc) & 15)
        return refuse(who, "tensors must be 16-byte aligned");
    if (hd != HD || nkv <= 0 || block_size <= 0) return refuse(who, "unsupported shape (head_dim must be 128)");
    if ((long)T * nkv >= 1L << 29) return refuse(who, "too many rows");
    return true;
}

RowsArgs rows_args(const int *slots, int T, int nkv, int block_size) {
    return RowsArgs{slots, T * nkv, nkv, page_div(nkv), page_div(block_size), head_bytes(block_size)};
}
// Workgroups for `rows` rows of K and of V at U rows a thread.
unsigned row_groups(int rows, int U) { return (unsigned)((2L * rows + U * ROWS_PER_PASS - 1) / (U * ROWS_PER_PASS)); }
// Four rows a thread once that still leaves four workgroups a CU.
int rows_a_thread(int rows) { return row_groups(rows, 4) >= 4u * llmgen_num_cus() ? 4 : 1; }

// ------------------------------------------------------------------------------------------------------------
// Split-K decode
// ------------------------------------------------------------------------------------------------------------
// One workgroup of 4 or 8 waves takes a span of one (sequence, kv head)'s visible keys, in tiles of 16 keys; a wave takes
// NT tiles (64 keys, 8.5 KB of codes and scales) a round and works alone until the end.
//   * K: lane (row l % 16, run l / 16) loads the 16 bytes that hold 32 values of one key, so a tile is one contiguous
//     kilobyte in one access, and converts them to four A fragments of v_mfma_f32_16x16x32_bf16 in registers.  Step c of
//     the product takes values 8c..8c+7 of every run; q is loaded in the same order, so no lane exchange is needed.
//     (The scaled fp8 x fp4 product would take the codes as they are, with q split exactly into two fp8 parts, but its
//     inner sums are kept to fewer bits: 9e-4 off on dot products of up to 59, where this one is exact to 2e-6.)
//   * S^T = K Q^T puts the tile's keys in rows (4 a lane) and the group's heads in columns, so the softmax over keys is
//     lane-local plus two lane exchanges, the running maximum and sum live in the lanes of their head, and two tiles'
//     probabilities, rounded to bf16 (off by at most 2^-8 of each, as in the other attention kernels), are the B fragment of
//     O^T = V^T P^T as they stand: the fragment's k-slots are assigned to keys in the order the accumulator holds them.
//   * V: lane l loads bytes 16 l of the tile (key l / 4, run l % 4), converts them and puts the bf16 row into the wave's
//     8 KB of LDS, from where ds_read_b64_tr_b16 reads it transposed.  Chunks of 16 bytes are swizzled by the row:
//     writes put 4 rows at once into chunks that differ in bits 2 and 3 only, reads take a pair of chunks of 8 rows, so
//     bits 0 and 1 of the swizzle differ among 4 rows, and bits 1 to 3 among 8.
//   * The loads of a round are issued when the registers they go to were just converted, a round ahead of their use.
// Measured: 16 sequences x 8 KV heads x 32768 keys (571 MB) 92 to 101 us, 5.7 to 6.2 TB/s, the rate of a read-only kernel;
// 32 ragged sequences of up to 1024 keys (20 MB) 9.2 us, where the chain table -> codes -> products -> merge counts.
// The waves' (m, l, O) are merged through LDS; a sequence with several spans leaves them in the caller's scratch, and
// the last workgroup of the (sequence, kv head) to finish merges them, by a counter that returns to 0.
constexpr int TILE = 16;  // keys a tile
constexpr int NT = 4;     // tiles a wave takes a round
constexpr int MAX_PARTS = 256;  // spans a sequence: their weights for 16 heads fill the 32 KB of LDS when merging

template <int NW>
struct DecodeLds {
    __attribute__((aligned(16))) unsigned char v[NW][32 * HD * 2];
    float m[NW][16];
    float l[NW][16];
    int last;
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
__device__ __forceinline__ s16x4_t ds_read_tr(const bf16_t *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)p);
}

__device__ __forceinline__ int swizzle(int row) { return (row & 7) | (row & 1) << 3; }

// maximum / sum over the four lanes l % 16 of a wave's 16-lane groups: swap the halves of every 32 lanes, then of 64
__device__ __forceinline__ float group_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t a = r[0], b = r[1];
    x = fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    auto t = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t c = t[0], d = t[1];
    return fmaxf(__builtin_bit_cast(float, c), __builtin_bit_cast(float, d));
}
__device__ __forceinline__ float group_sum(float x) {
    x += lane_xor(x, 16);
    return x + lane_xor(x, 32);
}

__device__ __forceinline__ u32x4_t ld16_stream(const void *p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_t *>(p));
}

// PAGE16: block_size % 16 == 0, a tile lies inside one page; else each lane looks its own key's page up.
template <bool PAGE16, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(3)))
    attn_decode_kv4_kernel(bf16_t *__restrict__ out, const bf16_t *__restrict__ q, const uint8_t *__restrict__ kc,
                           const uint8_t *__restrict__ vc, const int *__restrict__ block_tables,
                           const int *__restrict__ ctx_lens, const int *__restrict__ cu_q,
                           const int *__restrict__ tile_seq, int S, int nq, int nkv, int G, int max_blocks,
                           PageDiv div, float scale_log2, int window, int sinks, int span0, int nparts,
                           float *__restrict__ part_o, float *__restrict__ part_ml, int *__restrict__ counters) {
    __shared__ DecodeLds<NW> sm;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, rgrp = lane >> 4;
    const int kvh = blockIdx.x % nkv;
    const long rest = blockIdx.x / nkv;
    const int by = (int)(rest % S), part = (int)(rest / S);
    // a decode launch: `by` is the sequence and its row; a launch over a prefill step's tile list (cu_q): the single
    // rows of it, from the end of the list (longest first), one span each
    int s = by, row = by;
    if (cu_q) {
        s = tile_seq[S - 1 - by];
        row = cu_q[s];
        if (cu_q[s + 1] - row != 1) return;
    }
    const int block_size = div.bs;
    const int ctx = (int)min((long)ctx_lens[s], (long)max_blocks * block_size);
    if (ctx <= 0) {
        if (part == 0)
            for (int i = tid; i < G * HD / 2; i += 64 * NW)
                reinterpret_cast<uint32_t *>(out + ((long)row * nq + (long)kvh * G) * HD)[i] = 0;
        return;
    }
    // visible keys: [0, sinks) and [lo, ctx).  Tiles are counted over both: st tiles of sinks, then from lo's tile on.
    const int lo = max(0, ctx - window);
    const int lo_tile = lo / TILE;
    const int st = min((sinks + TILE - 1) / TILE, lo_tile);
    const int gap = (lo_tile - st) * TILE;
    const int nt = (ctx + TILE - 1) / TILE - (lo_tile - st);
    const int span = max(span0, ((nt + nparts - 1) / nparts + NT - 1) / NT * NT);  // tiles a workgroup
    const int np = (nt + span - 1) / span;
    if (part >= np) return;
    const int t_end = min(nt, (part + 1) * span);

    const long hb = head_bytes(block_size), page = hb * nkv;
    const int *bt = block_tables + (long)s * max_blocks;
    const uint8_t *kbase = kc + kvh * hb, *vbase = vc + kvh * hb;
    const long scale_at = (long)block_size * CODE_BYTES;

    // B operand: column col is head kvh * G + col (columns past G hold zeros and are never stored); step c holds values
    // rgrp * 32 + 8 c .. + 8
    bf16x8_t qf[4];
    {
        const bf16_t *qp = q + ((long)row * nq + (long)kvh * G + (col < G ? col : 0)) * HD + rgrp * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            u32x4_t x = ld16(qp + c * 8);
            if (col >= G) x = u32x4_t{0, 0, 0, 0};
            qf[c] = __builtin_bit_cast(bf16x8_t, x);
        }
    }
    f32x4_t o[8];  // O^T: dims db * 16 + rgrp * 4 + i of head col
#pragma unroll
    for (int db = 0; db < 8; ++db) o[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    u32x4_t kreg[NT], vreg[NT];
    uint32_t ksc[NT], vsc[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        kreg[i] = vreg[i] = u32x4_t{0, 0, 0, 0};
        ksc[i] = vsc[i] = 0;
    }
    auto tile_key = [&](int vt) { return vt * TILE + (vt >= st ? gap : 0); };
    auto hidden = [&](int t) -> bool { return (t >= ctx) | ((t < lo) & (t >= sinks)); };  // no branches
    // Pages are looked up ahead of use.  PAGE16: lane l holds the place of tile l % NT of round l / NT of the next AHEAD
    // rounds (looked up together, one load), read out as scalars; a tile past the span's end is its last one, read again
    // and masked, so that loads need no branch.  Else lanes hold the place of their own keys of the next round; a key
    // that is not visible is replaced by one that is.
    constexpr int AHEAD = 64 / NT;
    long at_codes = 0, at_scales = 0;
    long kcodes[NT], kscales[NT], vcodes[NT], vscales[NT];
    auto key_place = [&](int t, long &codes, long &scales) {
        const int blk = div(t), off = t - blk * block_size;
        const long base = (long)bt[blk] * page;
        codes = base + off * CODE_BYTES;
        scales = base + scale_at + off * SCALE_BYTES;
    };
    auto lookup = [&](int vt0, int r) {  // for round r of the wave, whose first tile is vt0
        if constexpr (PAGE16) {
            if (r % AHEAD == 0)
                key_place(tile_key(min(vt0 + (lane / NT) * NW * NT + lane % NT, t_end - 1)), at_codes, at_scales);
        } else {
            auto some = [&](int t) {
                t = min(t, ctx - 1);
                return t >= sinks && t < lo ? lo : t;
            };
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int t0 = tile_key(min(vt0 + i, t_end - 1));
                key_place(some(t0 + col), kcodes[i], kscales[i]);
                key_place(some(t0 + (lane >> 2)), vcodes[i], vscales[i]);
            }
        }
    };
    auto scalar = [](long x, int l) {
        const uint32_t a = __builtin_amdgcn_readlane((int)x, l), b = __builtin_amdgcn_readlane((int)(x >> 32), l);
        return (long)((uint64_t)b << 32 | a);
    };
    const int k_at = col * CODE_BYTES + rgrp * 16, ks_at = col * SCALE_BYTES + rgrp;
    auto load_k = [&](int r) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if constexpr (PAGE16) {
                const int l = r % AHEAD * NT + i;
                kreg[i] = ld16_stream(kbase + scalar(at_codes, l) + k_at);
                ksc[i] = (kbase + scalar(at_scales, l))[ks_at];
            } else {
                kreg[i] = ld16_stream(kbase + kcodes[i] + rgrp * 16);
                ksc[i] = kbase[kscales[i] + rgrp];
            }
        }
    };
    auto load_v = [&](int r) {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if constexpr (PAGE16) {
                const int l = r % AHEAD * NT + i;
                vreg[i] = ld16_stream(vbase + scalar(at_codes, l) + lane * 16);
                vsc[i] = (vbase + scalar(at_scales, l))[lane];
            } else {
                vreg[i] = ld16_stream(vbase + vcodes[i] + (lane & 3) * 16);
                vsc[i] = vbase[vscales[i] + (lane & 3)];
            }
        }
    };

    bf16_t *vl = reinterpret_cast<bf16_t *>(sm.v[wave]);
    int vt0 = part * span + wave * NT;
    if (vt0 < t_end) {
        lookup(vt0, 0);
        load_k(0);
        load_v(0);
        if (!PAGE16 && vt0 + NW * NT < t_end) lookup(vt0 + NW * NT, 1);
    }
    for (int r = 0; vt0 < t_end; vt0 += NW * NT, ++r) {
        const int next = vt0 + NW * NT;
        if (PAGE16 && next < t_end) lookup(next, r + 1);
        // ---- scores ----
        float sc[NT][4];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const float s2 = kv4_scale(ksc[i]);
            f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, kv4_to_bf16(kreg[i][c], s2)),
                                                              qf[c], acc, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) sc[i][j] = acc[j];
        }
        if (next < t_end) load_k(r + 1);
        // a round is visible as a whole except at the ends of the sinks, the window and the sequence (uniform)
        const int first = tile_key(vt0), end = tile_key(vt0 + NT - 1) + TILE;
        if (!(vt0 + NT <= t_end && end <= ctx && (vt0 >= st ? first >= lo : end <= sinks))) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const int t0 = tile_key(vt0 + i);
                const bool out_of_span = vt0 + i >= t_end;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    sc[i][j] = (out_of_span | hidden(t0 + rgrp * 4 + j)) ? -INFINITY : sc[i][j];
                // finite values behind a probability of 0
                vsc[i] = (out_of_span | hidden(t0 + (lane >> 2))) ? 0 : vsc[i];
            }
        }
        // ---- online softmax of head col.  Once every head has a reference m_run, probabilities are taken against it
        //      without a maximum (they may exceed 1: o / l is unchanged by a common factor); only a lane's sum beyond
        //      2^16 moves the reference (so a row's sum stays below 2^31 and values of 2^96 cannot overflow) ----
        u32x2_t p[NT];
        float lsum;
        auto probs = [&](float m_use) {
            lsum = 0.f;
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    e[j] = fast_exp2(__builtin_fmaf(sc[i][j], scale_log2, -m_use));
                    lsum += e[j];
                }
                p[i] = u32x2_t{pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3])};
            }
        };
        bool move = !__all(m_run > -INFINITY);
        if (!move) {
            probs(m_run);
            move = __any(!(lsum <= 0x1p16f));
        }
        if (move) {
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) mx = fmaxf(mx, sc[i][j]);
            const float m_new = fmaxf(m_run, group_max(mx) * scale_log2);  // scale > 0 commutes with the maximum
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            const float corr = fast_exp2(m_run - m_use);
            l_run *= corr;
#pragma unroll
            for (int db = 0; db < 8; ++db)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[db][j] *= corr;
            m_run = m_new;
            probs(m_use);
        }
        l_run += lsum;
        // ---- O^T += V^T P^T, two tiles (32 keys) a step ----
#pragma unroll
        for (int h = 0; h < NT / 2; ++h) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float s2 = kv4_scale(vsc[2 * h + i]);
                const int lr = i * 16 + (lane >> 2);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int chunk = ((lane & 3) * 4 + c) ^ swizzle(lr);
                    *reinterpret_cast<u32x4_t *>(vl + lr * HD + chunk * 8) = kv4_to_bf16(vreg[2 * h + i][c], s2);
                }
            }
            if (h == NT / 2 - 1 && next < t_end) {
                load_v(r + 1);
                if (!PAGE16 && next + NW * NT < t_end) lookup(next + NW * NT, r + 2);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            const u32x4_t pw = {p[2 * h][0], p[2 * h][1], p[2 * h + 1][0], p[2 * h + 1][1]};
            const bf16x8_t pb = __builtin_bit_cast(bf16x8_t, pw);
            const int tr = rgrp * 4 + (col >> 2);  // this lane's row of a transposed read, in either tile
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                const int chunk = (db * 2 + ((col & 3) >> 1)) ^ swizzle(tr);
                const bf16_t *src = vl + tr * HD + chunk * 8 + (col & 1) * 4;
                const s16x4_t a0 = ds_read_tr(src), a1 = ds_read_tr(src + 16 * HD);
                o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7)), pb, o[db], 0, 0,
                    0);
            }
            // the rows are overwritten next: keep every lane's reads ahead of those writes
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
    }

    // ---- merge the waves ----
    l_run = group_sum(l_run);
    if (rgrp == 0) {
        sm.m[wave][col] = m_run;
        sm.l[wave][col] = l_run;
    }
    if (col < G) {
        float *ow = reinterpret_cast<float *>(sm.v[wave]) + col * HD;
#pragma unroll
        for (int db = 0; db < 8; ++db) *reinterpret_cast<f32x4_t *>(ow + db * 16 + rgrp * 4) = o[db];
    }
    __syncthreads();
    for (int idx = tid; idx < G * HD; idx += 64 * NW) {
        const int g = idx / HD, d = idx % HD;
        float M = sm.m[0][g];
#pragma unroll
        for (int w = 1; w < NW; ++w) M = fmaxf(M, sm.m[w][g]);
        const float Mu = M == -INFINITY ? 0.f : M;
        float acc = 0.f, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float e = fast_exp2(sm.m[w][g] - Mu);
            acc += e * reinterpret_cast<const float *>(sm.v[w])[idx];
            L += e * sm.l[w][g];
        }
        const long h = (long)kvh * G + g;
        if (np == 1) {
            out[((long)row * nq + h) * HD + d] = __builtin_bit_cast(bf16_t, (__bf16)(acc / L));
        } else {  // device-coherent stores: another workgroup reads them
            const long slot = ((long)by * nq + h) * nparts + part;
            __hip_atomic_store(part_o + slot * HD + d, acc, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (d == 0) {
                __hip_atomic_store(part_ml + slot * 2, M, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                __hip_atomic_store(part_ml + slot * 2 + 1, L, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
        }
    }
    if (np == 1) return;

    // ---- merge the spans: every thread's stores are complete before the barrier, then one counter increment a
    //      workgroup elects the last, which reads the partials with device-coherent loads, in span order ----
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    int *cnt = counters + (long)by * nkv + kvh;
    if (tid == 0) sm.last = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == np - 1;
    __syncthreads();
    if (!sm.last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    auto ld = [](const float *x) { return __hip_atomic_load(x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
    float *ml = reinterpret_cast<float *>(sm.v);  // [head][span][m, l]
    const long slot0 = ((long)by * nq + (long)kvh * G) * nparts;
    for (int i = tid; i < G * np; i += 64 * NW) {
        const int g = i / np, p = i - g * np;
        const float *src = part_ml + (slot0 + (long)g * nparts + p) * 2;
        ml[2 * i] = ld(src);
        ml[2 * i + 1] = ld(src + 1);
    }
    __syncthreads();
    constexpr int MB = 16;  // partials a thread has in flight
    for (int idx = tid; idx < G * HD; idx += 64 * NW) {
        const int g = idx / HD, d = idx % HD;
        const float *mlg = ml + 2 * g * np;
        const float *po = part_o + (slot0 + (long)g * nparts) * HD + d;
        float M = -INFINITY, num = 0.f, den = 0.f;
        for (int p = 0; p < np; ++p) M = fmaxf(M, mlg[2 * p]);
        const float Mu = M == -INFINITY ? 0.f : M;
        for (int p0 = 0; p0 < np; p0 += MB) {
            float ov[MB];
#pragma unroll
            for (int j = 0; j < MB; ++j) ov[j] = p0 + j < np ? ld(po + (long)(p0 + j) * HD) : 0.f;
#pragma unroll
            for (int j = 0; j < MB; ++j)
                if (p0 + j < np) {
                    const float w = fast_exp2(mlg[2 * (p0 + j)] - Mu);
                    num += w * ov[j];
                    den += w * mlg[2 * (p0 + j) + 1];
                }
        }
        out[((long)row * nq + (long)kvh * G + g) * HD + d] = __builtin_bit_cast(bf16_t, (__bf16)(num / den));
    }
    if (tid == 0) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

struct DecodeShape {
    int S, nq, nkv, G, max_blocks, block_size;
    float sl2;
    int window, sinks;
};

void launch_decode(bf16_t *out, const bf16_t *q, const uint8_t *kc, const uint8_t *vc, const int *bt, const int *ctx,
                   const int *cu_q, const int *tile_seq, const DecodeShape &d, int span, int nparts, const Work &w,
                   int waves) {
    const long rows = (long)d.S * d.nq * nparts;
    float *part_o = nparts > 1 ? w.part : nullptr, *part_ml = nparts > 1 ? w.part + rows * HD : nullptr;
    auto go = [&](auto kern) {
        hipLaunchKernelGGL(kern, dim3((unsigned)((long)d.nkv * d.S * nparts)), dim3(64 * waves), 0, g_llmgen_stream, out, q,
                           kc, vc, bt, ctx, cu_q, tile_seq, d.S, d.nq, d.nkv, d.G, d.max_blocks, page_div(d.block_size),
                           d.sl2, d.window, d.sinks, span, nparts, part_o, part_ml, w.counters);
    };
    const bool page16 = d.block_size % TILE == 0;
    if (waves == 8) go(page16 ? attn_decode_kv4_kernel<true, 8> : attn_decode_kv4_kernel<false, 8>);
    else go(page16 ? attn_decode_kv4_kernel<true, 4> : attn_decode_kv4_kernel<false, 4>);
}

// The launch over d.S sequences (or entries of a tile list, `rows` of which have a single row), its keys split by this
// rule; false if the grid would be too large.
bool launch_split(bf16_t *out, const bf16_t *q, const uint8_t *kc, const uint8_t *vc, const int *bt, const int *ctx,
                  const int *cu_q, const int *tile_seq, const DecodeShape &d, int rows, int max_ctx, const Work &w) {
    // How the keys are split, measured over 1 to 64 sequences x 8 KV heads of 300 to 32768 keys: as few spans as leave no
    // CU idle, since each span more is one more partial result to merge.
    //   * enough (sequence, KV head) pairs for the chip: one span, of 8 waves up to two pairs a CU (256 pairs of 1500 keys
    //     12.6 us against 15.7 us with 4), of 4 above (512 pairs of 700 keys 11.6 against 14.5 us); from three quarters of
    //     a pair a CU on (192 pairs of 4096 keys 23.6 us, four spans of 4 waves 26.3 us; 128 pairs 23.2 and 19.5 us);
    //   * up to two rounds of 8 waves: one span (128 pairs of 700 keys 7.4 us against 12.0 us split, 8 pairs 7.2 and 7.7
    //     us), or three rounds from three eighths of a pair a CU on (96 pairs of 1500 keys 11.6 and 11.8 us, 64 pairs
    //     11.0 and 10.6 us);
    //   * else about two workgroups a CU, the spans a power of two (96 pairs of 4096 keys: 8 spans 16.6 us, 6 17.8 us; 112
    //     pairs: 4 spans 18.9 us, 8 21.0 us), of at least one round; 4 waves each, or 8 where that would be more than 8 spans (8 pairs of 32768 keys: 32 spans
    //     of 8 waves 15.8 us, 32 of 4 17.1 us; 8 pairs of 1500 keys: 6 spans of 4 waves 8.2 us, 3 of 8 9.2 us).
    long keys = std::max(1, std::min(max_ctx, d.max_blocks * d.block_size));
    keys = std::min(keys, (long)d.window + d.sinks + 2 * TILE);
    const long tiles = (keys + TILE - 1) / TILE, pairs = (long)rows * d.nkv, cus = llmgen_num_cus();
    const long rounds = (tiles + 8 * NT - 1) / (8 * NT);  // of 8 waves
    int waves = 8;
    long parts = 1;
    if (pairs >= 2 * cus) {
        waves = 4;
    } else if (pairs * 4 < 3 * cus && rounds > (pairs * 8 >= 3 * cus ? 3 : 2)) {
        while (2 * parts * pairs <= 3 * cus) parts *= 2;
        parts = std::min(parts, (tiles + 4 * NT - 1) / (4 * NT));
        if (parts > 8) parts = (parts + 1) / 2;
        else waves = 4;
    }
    parts = std::min<long>({parts, MAX_PARTS, w.floats / ((long)d.S * d.nq * (HD + 2))});
    if (parts < 1 || (long)d.S * d.nkv > WORK_COUNTERS) parts = 1;
    const long span = ((tiles + parts - 1) / parts + NT - 1) / NT * NT;
    if ((long)d.S * d.nkv * parts > 0x7fffffffL) return false;
    launch_decode(out, q, kc, vc, bt, ctx, cu_q, tile_seq, d, (int)span, (int)parts, w, waves);
    return true;
}

}  // namespace

extern "C" size_t hip_kv4_block_bytes(int nkv, int hd, int block_size) {
    if (hd != HD || nkv <= 0 || block_size <= 0) return 0;
    return (size_t)nkv * head_bytes(block_size);
}

extern "C" void hip_store_kv4(const bf16_t *k, const bf16_t *v, const int *slot_mapping, uint8_t *k_cache,
                              uint8_t *v_cache, int T, int nkv, int hd, int block_size) {
    if (T <= 0 || !check_rows("store_kv4", k, v, slot_mapping, k_cache, v_cache, T, nkv, hd, block_size)) return;
    const RowsArgs a = rows_args(slot_mapping, T, nkv, block_size);
    const int U = rows_a_thread(a.rows);
    hipLaunchKernelGGL(U == 4 ? store_kv4_kernel<4> : store_kv4_kernel<1>, dim3(row_groups(a.rows, U)), dim3(QUANT_THREADS), 0,
                       g_llmgen_stream, k, v, k_cache, v_cache, a);
}

extern "C" void hip_load_kv4(bf16_t *k, bf16_t *v, const int *slot_mapping, const uint8_t *k_cache,
                             const uint8_t *v_cache, int T, int nkv, int hd, int block_size) {
    if (T <= 0 || !check_rows("load_kv4", k, v, slot_mapping, k_cache, v_cache, T, nkv, hd, block_size)) return;
    const RowsArgs a = rows_args(slot_mapping, T, nkv, block_size);
    const int U = rows_a_thread(a.rows);
    hipLaunchKernelGGL(U == 4 ? load_kv4_kernel<4> : load_kv4_kernel<1>, dim3(row_groups(a.rows, U)), dim3(QUANT_THREADS), 0,
                       g_llmgen_stream, k, v, k_cache, v_cache, a);
}

extern "C" void hip_attn_decode_kv4(bf16_t *out, const bf16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                                    const int *block_tables, const int *ctx_lens, int S, int nq, int nkv, int hd,
                                    int max_blocks, int block_size, float scale, int window, int sinks, int max_ctx,
                                    void *work, size_t work_bytes) {
    const char *who = "attn_decode_kv4";
    if (S <= 0 || !check_attention(who, out, q, k_cache, v_cache, block_tables, ctx_lens, nq, nkv, hd, max_blocks,
                                   block_size, scale, window, sinks, work))
        return;
    DecodeShape d{S, nq, nkv, nq / nkv, max_blocks, block_size, scale * LLMGEN_LOG2E,
                  window ? std::min(window, NO_WINDOW) : NO_WINDOW, std::min(sinks, NO_WINDOW)};
    if (!launch_split(out, q, k_cache, v_cache, block_tables, ctx_lens, nullptr, nullptr, d, S, max_ctx,
                      split_work(work, work_bytes)))
        refuse(who, "too many sequences");
}

// The single rows of a prefill step over 4-bit pages (`rows` of them, as far as the caller knows).
bool llmgen_kv4_rows_of_prefill(bf16_t *out, const bf16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                                const int *block_tables, const int *ctx_lens, const int *cu_q, const int *tile_seq,
                                int n_tiles, int rows, int nq, int nkv, int max_blocks, int block_size, float scale_log2,
                                int window, int sinks, void *work, size_t work_bytes) {
    DecodeShape d{n_tiles, nq, nkv, nq / nkv, max_blocks, block_size, scale_log2, window, sinks};
    return launch_split(out, q, k_cache, v_cache, block_tables, ctx_lens, cu_q, tile_seq, d, rows, max_blocks * block_size,
                        split_work(work, work_bytes));
}
