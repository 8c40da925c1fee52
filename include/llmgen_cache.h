/*
 * llmgen_cache.h -- C-ABI of the other forms of the paged KV cache, in libllmgen_attn.so: pages held in 4 bits,
 * attention that keeps a sliding window and the first tokens, and page copies.  The reference engine has none of them
 * (its cache is bf16, its attention sees every key, its block manager in src/runner/block.zig neither shares nor moves
 * pages), so these entry points have no externs to replace.
 *
 * Conventions are those of llmgen_attn.h: device pointers unless named host, bf16 as uint16_t bits, launches on the
 * library stream, no allocation, no synchronisation, grids from integer arguments only (capturable).  Unsupported
 * arguments print one line to stderr, launch nothing and record hipErrorInvalidValue, which the next hip_last_error()
 * returns.  T, S, n_tiles and n of 0 or less are no-ops.
 */
#ifndef LLMGEN_CACHE_H
#define LLMGEN_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---------------------------------------------------------------------------------------------------------
 * Pages held in 4 bits
 *
 * A pool is [num_blocks][hip_kv4_block_bytes(nkv, hd, block_size)] bytes, 16-byte aligned.  A page holds, for each KV
 * head in turn, block_size rows of 64 code bytes (128 e2m1 values, the even one in the low half of its byte), then
 * block_size rows of 4 scale bytes, padded to a multiple of 16 bytes together.  A code is a sign bit above an index into
 * 0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale byte b stands for 2^(b - 127), 255 for NaN; a scale covers 32 consecutive values
 * of a row (the layout of the OCP microscaling formats with a block of 32 along the head).
 *
 * Writing x: the block's exponent is e = floor(log2 amax) - 2, one more where amax > 7 * 2^e (so that no value of the
 * block is off by more than 2^e, half the grid's last step), at least -127 and at most 125; the code is |x| / 2^e rounded
 * to the nearest grid value, ties to the even index, 6 beyond it.  A block of zeros has scale byte 0; a block with an
 * infinity or NaN has scale byte 255 and codes 0: all its values are NaN.  Every step is exact, so the bytes are
 * defined bit for bit.  hd must be 128.
 * ------------------------------------------------------------------------------------------------------- */

/* Bytes of one page of a K or V pool; 0 for an unsupported shape. */
size_t hip_kv4_block_bytes(int nkv, int hd, int block_size);

/* k, v [T, nkv, hd] bf16, 16-byte aligned -> the pages at slot_mapping[t] (block = slot / block_size, offset = slot %
 * block_size), as hip_store_kv; slot < 0 rows are skipped.  Rows that share a slot leave one of them, not told which. */
void hip_store_kv4(const uint16_t *k, const uint16_t *v, const int32_t *slot_mapping, uint8_t *k_cache,
                   uint8_t *v_cache, int T, int nkv, int hd, int block_size);

/* The rows at slot_mapping[t] as the bf16 values they stand for, into k, v [T, nkv, hd]; rows of slot < 0 are left as
 * they are.  Exact for every page that hip_store_kv4 wrote (a value is a grid value times a power of two). */
void hip_load_kv4(uint16_t *k, uint16_t *v, const int32_t *slot_mapping, const uint8_t *k_cache,
                  const uint8_t *v_cache, int T, int nkv, int hd, int block_size);

/* ---------------------------------------------------------------------------------------------------------
 * Attention over 4-bit pages, and with a sliding window and sinks over either kind of page
 *
 * A query row at position p sees the keys k <= p with k > p - window or k < sinks: the last `window` positions, its own
 * among them, and the first `sinks` ones.  window 0: no window, every key k <= p (sinks is then ignored).  window and
 * sinks are at least 0.  Pages and block-table entries that hold no key that some row sees are not read, so a host may
 * free the pages between the sinks and the window.  Values in places that a row does not see do not reach it, infinities
 * and NaN among them.
 *
 * out, q [T, nq, hd] bf16; hd == 128, nq / nkv in {1, 2, 4, 8, 16}, scale > 0 and finite.  Softmax statistics and sums
 * are f32; probabilities are rounded to bf16 for the matrix cores.  Sums are taken against a running reference and
 * divided at the end: values of up to 2^96 cannot overflow them, beyond that a result may be infinite.
 *
 * work is the calls' scratch: hip_attn_work_bytes() bytes of device memory (16-byte aligned), set up once by
 * hip_attn_work_init and left ready by every call.  Calls that may run at the same time (two streams, two graphs
 * replayed on two streams) need one each; calls on one stream share one.  With less memory, or NULL, calls that would
 * split a sequence's keys over workgroups do so less, or not at all; results then differ in their last bits.
 * ------------------------------------------------------------------------------------------------------- */
size_t hip_attn_work_bytes(void);
/* Enqueues the clearing of the scratch's counters (a kernel: it may be captured). */
void hip_attn_work_init(void *work, size_t work_bytes);

/* One query row a sequence: q, out [S, nq, hd]; block_tables [S, max_blocks]; ctx_lens[s] = cached keys, the row's own
 * among them (its position is ctx - 1).  ctx <= 0 rows output 0.  max_ctx is the longest context the caller expects and
 * steers only how the keys are split: longer ones (up to max_blocks * block_size) are attended in full. */
void hip_attn_decode_window(uint16_t *out, const uint16_t *q, const uint16_t *k_cache, const uint16_t *v_cache,
                            const int32_t *block_tables, const int32_t *ctx_lens, int S, int nq, int nkv, int hd,
                            int max_blocks, int block_size, float scale, int window, int sinks, int max_ctx, void *work,
                            size_t work_bytes);
void hip_attn_decode_kv4(uint16_t *out, const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                         const int32_t *block_tables, const int32_t *ctx_lens, int S, int nq, int nkv, int hd,
                         int max_blocks, int block_size, float scale, int window, int sinks, int max_ctx, void *work,
                         size_t work_bytes);

/* Causal varlen rows, with the metadata of hip_attn_prefill: sequence s owns rows [cu_q[s], cu_q[s+1]), ctx_lens[s] =
 * keys after this step, tile_seq / tile_q0 [n_tiles] list the query tiles of hip_attn_prefill_tile() rows, in any order
 * (llmgen_fill_meta's is fastest).  Sequences with ctx < q_len are padding: rows of 0; rows behind the last sequence are
 * not written.  single_rows as in hip_attn_prefill_rows: the number of sequences with one row; 0 none, negative
 * unknown.  Single rows are streamed by a decode launch unless the count is 0, their keys split as there; a wrong count
 * costs time only. */
void hip_attn_prefill_window(uint16_t *out, const uint16_t *q, const uint16_t *k_cache, const uint16_t *v_cache,
                             const int32_t *block_tables, const int32_t *ctx_lens, const int32_t *cu_q,
                             const int32_t *tile_seq, const int32_t *tile_q0, int n_tiles, int nq, int nkv, int hd,
                             int max_blocks, int block_size, float scale, int window, int sinks, int single_rows,
                             void *work, size_t work_bytes);
void hip_attn_prefill_kv4(uint16_t *out, const uint16_t *q, const uint8_t *k_cache, const uint8_t *v_cache,
                          const int32_t *block_tables, const int32_t *ctx_lens, const int32_t *cu_q,
                          const int32_t *tile_seq, const int32_t *tile_q0, int n_tiles, int nq, int nkv, int hd,
                          int max_blocks, int block_size, float scale, int window, int sinks, int single_rows,
                          void *work, size_t work_bytes);

/* ---------------------------------------------------------------------------------------------------------
 * Page copies
 *
 * Copies page src[i] onto page dst[i] in each of n_pools pools (the K and V pools of every layer, of either kind of
 * page).  pools, src and dst are host arrays, read before the call returns (a captured call keeps what they held): pools
 * holds device pointers (16-byte aligned), the pages are num_blocks x block_bytes (a multiple of 16, at most 2^28).
 * Every id must lie in [0, num_blocks), no page may be the destination of two pairs, and none both a source and a
 * destination (src[i] == dst[i] is a pair that does nothing): the pairs then have no order.  Otherwise nothing is copied.
 * ------------------------------------------------------------------------------------------------------- */
void hip_copy_blocks(void *const *pools, int n_pools, size_t block_bytes, int num_blocks, const int32_t *src,
                     const int32_t *dst, int n);

#ifdef __cplusplus
}
#endif

#endif /* LLMGEN_CACHE_H */
