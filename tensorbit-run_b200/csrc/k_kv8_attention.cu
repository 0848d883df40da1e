// k_kv8_attention.cu -- attention of Q rows over the paged 8-bit cache.
//
// out = sum_j p_j v_j, p = softmax(scale q.k_j) over the keys a row sees, with
// k_j = code * scale of the page.  A CTA per (row, head): each warp walks
// every fourth key with the lanes across the head dimension, a running max m,
// sum l and weighted v of its own (m' = max(m, s): l and v scaled by
// exp(m - m')), and the warps' states are joined at the end.
#include "kv8.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

struct Args {
    kv8::Batch b;
    const void* q;
    void* out;
    float* lse;
    int64_t q_stride, out_stride;
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    unsigned* status;
    float scale;
    int hq, hkv, d, window, max_rows, max_len;
};

template <typename T, int FORMAT>
__global__ void __launch_bounds__(kThreads) k_attention(const __grid_constant__ Args a) {
    __shared__ float part[kWarps][kv8::kMaxDim];
    __shared__ float pm[kWarps], pl[kWarps];
    const kv8::Batch& b = a.b;
    const int row = blockIdx.x, head = blockIdx.y, g = head / (a.hq / a.hkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int lo = 0, hi = b.n_seqs - 1;  // the last sequence that starts at or before the row
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (b.row_start[mid] <= row)
            lo = mid;
        else
            hi = mid - 1;
    }
    const kv8::Seq s = kv8::sequence(b, lo);
    if (row < s.lo || row >= s.lo + s.n) return;  // nobody's
    const bool ok = s.len <= a.max_len && s.n <= a.max_rows &&
                    s.len <= ((int64_t)b.width << b.page_shift);
    if (!ok && threadIdx.x == 0) atomicOr(a.status, TB_B200_FLAG_POSITION_RANGE);
    const int p = ok ? s.first + row - s.lo : -1;
    const int j0 = a.window ? max(p - a.window + 1, 0) : 0;
    const T* q = static_cast<const T*>(a.q) + row * a.q_stride + (int64_t)head * a.d;
    float qv[8], acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        qv[i] = lane + 32 * i < a.d ? tbk::Elt<T>::load(q + lane + 32 * i) : 0.0f;
        acc[i] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    for (int j = j0 + warp; j <= p; j += kWarps) {
        const int id = b.table[lo * b.table_stride + (j >> b.page_shift)];
        if (id < 0 || id >= b.n_pages) {
            if (lane == 0) atomicOr(a.status, TB_B200_FLAG_PAGE_RANGE);
            continue;
        }
        const int64_t unit = (int64_t)id * a.hkv + g;
        const int64_t at = ((unit << b.page_shift) + (j & ((1 << b.page_shift) - 1))) * a.d;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < a.d)
                dot = fmaf(qv[i], kv8::decode<FORMAT>(a.k[at + lane + 32 * i]), dot);
        const float sc = tbk::warp_sum(dot) * a.k_scale[unit] * a.scale;
        const float mn = fmaxf(m, sc), keep = expf(m - mn), e = expf(sc - mn);
        const float ev = e * a.v_scale[unit];
        l = l * keep + e;
        m = mn;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < a.d)
                acc[i] = fmaf(ev, kv8::decode<FORMAT>(a.v[at + lane + 32 * i]), acc[i] * keep);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < a.d) part[warp][lane + 32 * i] = acc[i];
    if (lane == 0) {
        pm[warp] = m;
        pl[warp] = l;
    }
    __syncthreads();
    float top = -INFINITY, sum = 0.0f, w[kWarps];
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, pm[i]);
    for (int i = 0; i < kWarps; ++i) {
        w[i] = pm[i] == -INFINITY ? 0.0f : expf(pm[i] - top);
        sum += w[i] * pl[i];
    }
    T* out = static_cast<T*>(a.out) + row * a.out_stride + (int64_t)head * a.d;
    for (int i = threadIdx.x; i < a.d; i += kThreads) {
        float y = 0.0f;
        for (int k = 0; k < kWarps; ++k) y += w[k] * part[k][i];
        tbk::Elt<T>::store(out + i, sum == 0.0f ? 0.0f : y / sum);
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[(int64_t)row * a.hq + head] = sum == 0.0f ? -INFINITY : top + logf(sum);
}

int check(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, const TbB200Kv8Attention* t,
          bool pointers) {
    int rc = kv8::check_cache(cache, pointers);
    if (rc == TB_OK) rc = kv8::check_batch(batch, pointers);
    if (rc != TB_OK) return rc;
    if (!t) return TB_ERR_INVALID_ARG;
    if (t->dtype != TB_DTYPE_F32 && t->dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    if (t->n_heads < 1 || t->n_heads > 65535 || t->n_heads % cache->n_kv_heads ||
        t->window < 0 || t->max_rows < 0 || t->max_len < 0)
        return TB_ERR_INVALID_SHAPE;
    const int64_t width = (int64_t)t->n_heads * cache->head_dim;
    if (batch->rows > 1 && pointers && (t->q_stride < width || t->out_stride < width))
        return TB_ERR_INVALID_SHAPE;
    if (pointers && batch->rows && batch->n_seqs && (!t->q || !t->out || t->q == t->out))
        return TB_ERR_INVALID_ARG;
    return TB_OK;
}

}  // namespace

extern "C" int tb_b200_kv8_attention_workspace(const TbB200Kv8* cache,
                                               const TbB200Kv8Batch* batch,
                                               const TbB200Kv8Attention* attention,
                                               size_t* bytes) {
    const int rc = check(cache, batch, attention, false);
    if (rc != TB_OK) return rc;
    if (!bytes) return TB_ERR_INVALID_ARG;
    *bytes = 0;
    return TB_OK;
}

extern "C" int tb_b200_kv8_attention(const TbB200Kv8* cache, const TbB200Kv8Batch* batch,
                                     const TbB200Kv8Attention* attention, void* stream) {
    const TbB200Kv8Attention* t = attention;
    const int rc = check(cache, batch, t, true);
    if (rc != TB_OK) return rc;
    if (batch->rows == 0 || batch->n_seqs == 0) return TB_OK;
    tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    const Args a = {kv8::view(cache, batch),
                    t->q,
                    t->out,
                    t->lse,
                    t->q_stride,
                    t->out_stride,
                    static_cast<const uint8_t*>(cache->k),
                    static_cast<const uint8_t*>(cache->v),
                    cache->k_scale,
                    cache->v_scale,
                    ds->status,
                    t->scale,
                    t->n_heads,
                    cache->n_kv_heads,
                    cache->head_dim,
                    t->window,
                    t->max_rows,
                    t->max_len};
    const dim3 grid((unsigned)batch->rows, (unsigned)t->n_heads);
    cudaStream_t s = tbh::stream_of(stream);
    const bool f32 = t->dtype == TB_DTYPE_F32, int8 = cache->format == kv8::kInt8;
    if (f32 && int8)
        k_attention<float, kv8::kInt8><<<grid, kThreads, 0, s>>>(a);
    else if (f32)
        k_attention<float, kv8::kE4m3><<<grid, kThreads, 0, s>>>(a);
    else if (int8)
        k_attention<__nv_bfloat16, kv8::kInt8><<<grid, kThreads, 0, s>>>(a);
    else
        k_attention<__nv_bfloat16, kv8::kE4m3><<<grid, kThreads, 0, s>>>(a);
    TB_LAUNCH_CHECK("8-bit cache attention kernel");
    return TB_OK;
}
