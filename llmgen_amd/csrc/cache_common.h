// cache_common.h -- what the kernels on the other forms of the paged cache share: the layout of a 4-bit page, the set of
// keys a sliding window with sinks leaves visible, the caller's scratch, and the checks of their launchers.
#pragma once
#include "hip_common.h"
#include "llmgen_cache.h"

#include <math.h>

namespace llmgen_cache {

constexpr int HD = 128;
constexpr int CODE_BYTES = HD / 2;    // codes of a row
constexpr int SCALE_BYTES = HD / 32;  // scales of a row

// Bytes one KV head takes in a 4-bit page: the rows' codes, then their scales padded to 16 bytes, so that every page
// and head starts on a 16-byte boundary whatever the block size.
__host__ __device__ __forceinline__ long head_bytes(int block_size) {
    return (long)block_size * CODE_BYTES + (((long)block_size * SCALE_BYTES + 15) & ~15L);
}

// 8 codes of a word -> 8 bf16 (two per instruction), times the power of two in the exponent field of `scale`
__device__ __forceinline__ u32x4_t kv4_to_bf16(uint32_t w, float scale) {
    u32x4_t r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3));
    return r;
}
// the f32 whose exponent field is scale byte b (0 gives the subnormal field that the conversion reads as 2^-127)
__device__ __forceinline__ float kv4_scale(uint32_t b) { return __builtin_bit_cast(float, b << 23); }

// Writing: the magnitude bits of the largest of 8 bf16 values (they order as the values do, infinities and NaN above all)
__device__ __forceinline__ uint32_t kv4_top(u32x4_t x) {
    const uint32_t x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
    return max(max(max(x0 & 0x7fffu, x0 >> 16 & 0x7fffu), max(x1 & 0x7fffu, x1 >> 16 & 0x7fffu)),
               max(max(x2 & 0x7fffu, x2 >> 16 & 0x7fffu), max(x3 & 0x7fffu, x3 >> 16 & 0x7fffu)));
}
// The scale byte of a run whose largest value has the magnitude bits `top`.  floor(log2 amax) is the exponent field for
// normal numbers.  Subnormal ones have an amax below 2^-126, and e would fall below -127 for any amax under 2^-125: both
// take the clamp.  Mantissas above 1.75 (0x60 of 7 bits) round up.
__device__ __forceinline__ int kv4_scale_byte(uint32_t top) {
    const int byte = (int)(top >> 7) - 2 + ((top & 0x7f) > 0x60 ? 1 : 0);
    return top >= 0x7f80u ? 255 : top == 0 ? 0 : min(max(byte, 0), 252);
}
// 8 bf16 values of a run with that scale byte -> 8 codes
__device__ __forceinline__ uint32_t kv4_codes(u32x4_t x, int byte) {
    const uint32_t x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];
    const float s = kv4_scale(byte == 255 ? 127 : byte);
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x0), s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x1), s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x2), s, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf16x2_t, x3), s, 3);
    return byte == 255 ? 0 : w;
}

// Division of a token's position by the block size: a shift for a power of two, else a multiplication by
// floor(2^32 / bs), which falls short by at most one for positions below 2^30.
struct PageDiv {
    int bs, shift;
    uint32_t magic;
    __device__ __forceinline__ int operator()(int t) const {
        if (shift >= 0) return t >> shift;
        const int d = (int)__umulhi((uint32_t)t, magic);
        return t - d * bs >= bs ? d + 1 : d;
    }
};
inline PageDiv page_div(int bs) {
    return PageDiv{bs, (bs & (bs - 1)) == 0 ? __builtin_ctz(bs) : -1, bs > 1 ? (uint32_t)((1ull << 32) / bs) : 0u};
}

// No window is a window longer than any sequence, so that the kernels know one rule only.
constexpr int NO_WINDOW = 1 << 30;

// The caller's scratch: counters (0 between launches), then partial results.
constexpr int WORK_COUNTERS = 1 << 14;
constexpr size_t WORK_HEAD = WORK_COUNTERS * sizeof(int);
struct Work {
    int *counters = nullptr;
    float *part = nullptr;
    long floats = 0;  // room for partial results
};
inline Work split_work(void *work, size_t bytes) {
    Work w;
    if (!work || bytes <= WORK_HEAD) return w;
    w.counters = static_cast<int *>(work);
    w.part = reinterpret_cast<float *>(static_cast<char *>(work) + WORK_HEAD);
    w.floats = (long)((bytes - WORK_HEAD) / sizeof(float));
    return w;
}

inline bool refuse(const char *who, const char *what) {
    fprintf(stderr, "[llmgen-hip] %s: %s\n", who, what);
    llmgen_record_error(hipErrorInvalidValue);
    return false;
}

// The checks the four attention entry points share; true if the call can be launched.
inline bool check_attention(const char *who, const void *out, const void *q, const void *kc, const void *vc,
                            const void *bt, const void *ctx, int nq, int nkv, int hd, int max_blocks, int block_size,
                            float scale, int window, int sinks, const void *work) {
    if (!out || !q || !kc || !vc || !bt || !ctx) return refuse(who, "a tensor is missing");
    if (((uintptr_t)out | (uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)work) & 15)
        return refuse(who, "tensors and scratch must be 16-byte aligned");
    if (hd != HD) return refuse(who, "only head_dim=128 is supported");
    if (nkv <= 0 || nq <= 0 || nq % nkv != 0) return refuse(who, "bad head counts");
    const int G = nq / nkv;
    if (G != 1 && G != 2 && G != 4 && G != 8 && G != 16) return refuse(who, "unsupported GQA group size");
    if (max_blocks <= 0 || block_size <= 0 || (long)max_blocks * block_size > 0x3fffffffL)
        return refuse(who, "bad block table shape (at most 2^30 - 1 tokens a sequence)");
    if (!(scale > 0.f) || isinf(scale)) return refuse(who, "scale must be positive and finite");
    if (window < 0 || sinks < 0) return refuse(who, "window and sinks must not be negative");
    return true;
}

}  // namespace llmgen_cache

// Internal: the single rows (segments with one query row, `rows` of them as far as the caller knows) of a prefill step
// over 4-bit pages; defined in kv4.hip, launched by hip_attn_prefill_kv4.  window is NO_WINDOW where there is none.
// False if the grid would be too large.
__attribute__((visibility("hidden"))) bool llmgen_kv4_rows_of_prefill(
    bf16_t *out, const bf16_t *q, const uint8_t *k_cache, const uint8_t *v_cache, const int *block_tables,
    const int *ctx_lens, const int *cu_q, const int *tile_seq, int n_tiles, int rows, int nq, int nkv, int max_blocks,
    int block_size, float scale_log2, int window, int sinks, void *work, size_t work_bytes);
