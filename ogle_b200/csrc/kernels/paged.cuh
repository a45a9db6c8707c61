// The paged 8-bit key/value cache: what its kernels share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace ogle {
namespace paged {

// OglePagedBatch as the kernels take it, the page size as a shift.
struct Batch {
    int n_seqs, n_rows, max_rows, max_kv_len;
    int q_heads, kv_heads, group, dim;
    int page_shift, n_pages, table_stride;
    int dtype;
    long long page_stride, head_stride, token_stride;
    const int *row_start, *kv_len, *block_table;
    unsigned char *k_cache, *v_cache;
    float *k_scale, *v_scale;
};

// Checks what the host can see and translates it. OGLE_OK with out.n_seqs 0 where there is nothing to do.
inline int translate(const OglePagedBatch* b, Batch& out) {
    if (!b || b->n_seqs < 0 || b->n_rows < 0 || b->max_rows < 0 || b->max_kv_len < 0) return OGLE_ERR_INVALID;
    if (b->dtype < OGLE_F32 || b->dtype > OGLE_BF16) return OGLE_ERR_INVALID;
    if (b->kv_heads < 1 || b->q_heads < 1 || b->q_heads % b->kv_heads != 0 || b->kv_heads > 4096 || b->q_heads > 65536) return OGLE_ERR_INVALID;
    if (b->head_dim < 16 || b->head_dim % 16 != 0) return OGLE_ERR_INVALID;
    if (b->head_dim > 256) return OGLE_ERR_UNSUPPORTED;
    if (b->page_tokens < 16 || b->page_tokens > 1024 || (b->page_tokens & (b->page_tokens - 1)) != 0) return OGLE_ERR_INVALID;
    if (b->n_pages < 0 || b->table_stride < 0 || b->n_seqs > (1 << 24)) return OGLE_ERR_INVALID;
    // rows x heads and tokens are counted in 32 bits
    if ((long long)b->n_rows * b->q_heads > (1LL << 30) || b->max_kv_len > (1 << 30)) return OGLE_ERR_UNSUPPORTED;
    if ((b->page_stride | b->head_stride | b->token_stride) & 15) return OGLE_ERR_ALIGNMENT;
    if (b->page_stride < 1 || b->head_stride < 1 || b->token_stride < b->head_dim) return OGLE_ERR_INVALID;
    out = Batch{};
    if (b->n_seqs == 0 || b->n_rows == 0) return OGLE_OK;
    if (!b->kv_len || !b->block_table || !b->k_cache || !b->v_cache || !b->k_scale || !b->v_scale) return OGLE_ERR_INVALID;
    if (!b->row_start && (b->n_rows != b->n_seqs || b->max_rows < 1)) return OGLE_ERR_INVALID;
    // no sequence is longer than its row of the table
    if (b->max_kv_len > (long long)b->table_stride * b->page_tokens) return OGLE_ERR_INVALID;
    if (!aligned16(b->k_cache) || !aligned16(b->v_cache)) return OGLE_ERR_ALIGNMENT;
    int shift = 4;
    while ((1 << shift) < b->page_tokens) ++shift;
    out.n_seqs = b->n_seqs; out.n_rows = b->n_rows; out.max_rows = b->max_rows; out.max_kv_len = b->max_kv_len;
    out.q_heads = b->q_heads; out.kv_heads = b->kv_heads; out.group = b->q_heads / b->kv_heads; out.dim = b->head_dim;
    out.page_shift = shift; out.n_pages = b->n_pages; out.table_stride = b->table_stride; out.dtype = b->dtype;
    out.page_stride = b->page_stride; out.head_stride = b->head_stride; out.token_stride = b->token_stride;
    out.row_start = b->row_start; out.kv_len = b->kv_len; out.block_table = b->block_table;
    out.k_cache = static_cast<unsigned char*>(b->k_cache); out.v_cache = static_cast<unsigned char*>(b->v_cache);
    out.k_scale = b->k_scale; out.v_scale = b->v_scale;
    return OGLE_OK;
}

// Whether activations at p with these strides (elements) can be read 16 bytes at a time.
inline bool strides_ok(const void* p, long long row, long long head, int dtype) {
    const int size = dtype == OGLE_F32 ? 4 : 2;
    return aligned16(p) && (row * size) % 16 == 0 && (head * size) % 16 == 0;
}

// One sequence: rows [row0, row0 + n) of the call, of which the first stands at position `first` (below 0: before the text), and len tokens.
struct Sequence { int row0, n, len, first; };

// What the device holds, cut to the bounds that the host gave: nothing outside the buffers is named whatever is in it. Rows keep the
// positions that the whole counts give them.
__device__ __forceinline__ Sequence sequence(const Batch& a, int b) {
    Sequence s;
    s.row0 = a.row_start ? a.row_start[b] : b;
    const int end = a.row_start ? a.row_start[b + 1] : b + 1;
    s.len = max(a.kv_len[b], 0);
    s.row0 = min(max(s.row0, 0), a.n_rows);
    s.n = min(max(end, s.row0), a.n_rows) - s.row0;
    s.first = s.len - s.n;
    s.len = min(s.len, a.max_kv_len);
    s.n = min(s.n, a.max_rows);
    return s;
}

// The page of token block `i` of sequence b, or -1.
__device__ __forceinline__ int page_of(const Batch& a, int b, int i) {
    const int p = __ldg(a.block_table + (long long)b * a.table_stride + i);
    return (unsigned)p < (unsigned)a.n_pages ? p : -1;
}

__device__ __forceinline__ float to_float(const void* p, long long i, int dtype) {
    if (dtype == OGLE_F32) return static_cast<const float*>(p)[i];
    if (dtype == OGLE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Two e4m3 bytes (the low one first) as two fp16, exactly.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
// Four of them: the lower two, the upper two.
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t v, uint32_t& lower, uint32_t& upper) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
        : "=r"(lower), "=r"(upper) : "r"(v));
}
// Two fp32 as e4m3, round to nearest even, beyond 448 the largest value, NaN as NaN.
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

}  // namespace paged
}  // namespace ogle
