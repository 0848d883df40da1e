// kv8.cuh -- what the kernels of the paged 8-bit KV cache share: the checked
// view of a cache and a batch, and the codes.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <stdint.h>

#include "tb_device.cuh"
#include "tb_internal.h"

namespace kv8 {

constexpr int kInt8 = TB_B200_KV_INT8, kE4m3 = TB_B200_KV_E4M3;
constexpr int kMaxDim = 256;

// A batch as the kernels see it.
struct Batch {
    const int32_t *row_start, *lengths, *table;
    int64_t table_stride;
    int n_seqs, width, page_shift;
    int rows;
    int64_t n_pages;
};

// Rows [lo, lo + n) of sequence i and the position of the first.  Malformed
// row_start values are clamped into the buffers.
struct Seq {
    int lo, n, len, first;
};

__device__ __forceinline__ Seq sequence(const Batch& b, int i) {
    Seq s;
    s.lo = min(max(b.row_start[i], 0), b.rows);
    s.n = max(min(max(b.row_start[i + 1], 0), b.rows) - s.lo, 0);
    s.len = max(b.lengths[i], 0);
    s.first = s.len - s.n;
    return s;
}

// The last sequence whose first slot, start(row_start, i), is at or before `slot`,
// by a whole warp, 32 candidates at a time; s: its rows.  The first one if there is
// none.
template <typename F>
__device__ __forceinline__ int find_sequence(const Batch& b, int slot, F start, Seq& s) {
    const int lane = threadIdx.x & 31;
    int seq = 0;
    for (int n = b.n_seqs;;) {  // it is in [seq, seq + n)
        const int step = (n + 31) / 32, i = min(seq + lane * step, b.n_seqs - 1);
        const Seq mine = sequence(b, i);  // of the last look, the answer's too
        const bool before = lane * step < n && start(mine.lo, i) <= slot;
        const int last = 31 - __clz(__ballot_sync(tbk::kFull, before) | 1);
        seq += last * step;
        n = min(step, n - last * step);
        if (step > 1) continue;
        s.lo = __shfl_sync(tbk::kFull, mine.lo, last);
        s.n = __shfl_sync(tbk::kFull, mine.n, last);
        s.len = __shfl_sync(tbk::kFull, mine.len, last);
        s.first = s.len - s.n;
        return seq;
    }
}

// The first key that a row at position p attends.
__device__ __forceinline__ int first_seen(int p, int window) {
    return window && p >= window ? p - window + 1 : 0;
}

// The cache's pointers and shapes, checked: TB_OK or the error to return.
inline int check_cache(const TbB200Kv8* c, bool pointers) {
    if (!c) return TB_ERR_INVALID_ARG;
    if (c->format != kInt8 && c->format != kE4m3) return TB_ERR_UNSUPPORTED_DTYPE;
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        return TB_ERR_INVALID_SHAPE;
    if (c->n_kv_heads < 1 || c->n_kv_heads > 65535 || c->head_dim < 16 ||
        c->head_dim > kMaxDim || c->head_dim % 16 || c->n_pages < 1 ||
        c->n_pages > INT32_MAX / c->n_kv_heads)
        return TB_ERR_INVALID_SHAPE;
    if (pointers &&
        (!c->k || !c->v || !c->k_scale || !c->v_scale || !tbh::aligned16(c->k) ||
         !tbh::aligned16(c->v)))
        return TB_ERR_INVALID_ARG;
    return TB_OK;
}

inline int check_batch(const TbB200Kv8Batch* b, bool pointers) {
    if (!b) return TB_ERR_INVALID_ARG;
    if (b->n_seqs < 0 || b->n_seqs > 65535 || b->rows < 0 || b->rows > INT32_MAX / 2 ||
        b->table_width < 0 || b->table_stride < b->table_width)
        return TB_ERR_INVALID_SHAPE;
    if (pointers && b->n_seqs && b->rows &&
        (!b->row_start || !b->lengths || (b->table_width && !b->page_table)))
        return TB_ERR_INVALID_ARG;
    return TB_OK;
}

inline Batch view(const TbB200Kv8* c, const TbB200Kv8Batch* b) {
    int shift = 4;
    while ((1 << shift) < c->page) ++shift;
    return {b->row_start, b->lengths,     b->page_table,  b->table_stride, b->n_seqs,
            b->table_width, shift, (int)b->rows, c->n_pages};
}

// Attention of many rows a sequence (k_kv8_chunk.cu): whether a call's bounds
// suit it, and the call, checked before.
bool chunk_suits(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
                 int sm_count);
int chunk_attention(const TbB200Kv8* cache, const TbB200Kv8Batch* batch,
                    const TbB200Kv8Attention* t, cudaStream_t stream);

// ------------------------------------------------------------------ codes
// A code's value, and the nearest code (ties to even) of a value within
// the format's range.
template <int FORMAT>
__device__ __forceinline__ float decode(uint8_t c) {
    if constexpr (FORMAT == kInt8) {
        return (float)(int8_t)c;
    } else {
        // sign, 4 exponent and 3 mantissa bits sit in f16's places two binades
        // of bias (2^8) below their value, subnormals included
        const uint16_t h = (uint16_t)((c & 0x80) << 8 | (c & 0x7f) << 7);
        return __half2float(__ushort_as_half(h)) * 256.0f;
    }
}

template <int FORMAT>
__device__ __forceinline__ uint8_t encode(float x) {
    if constexpr (FORMAT == kInt8)
        return (uint8_t)(int8_t)__float2int_rn(x);
    else
        return (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}

}  // namespace kv8
