// k_kv8_append.cu -- K and V rows into the paged 8-bit cache.
//
// A page of one head keeps one scale, so the rows a call adds to it are
// handled together: amax over them, s = the least power of two with amax <=
// MAX s (not below 2^-100, not below the scale of earlier tokens), the earlier
// codes rescaled where s grew, the new codes rne(x / s).  With s a power of two
// x / s is exact, so a code depends on nothing but its definition, and a
// rescaling by 2^-k adds at most half a step that every later one halves; a
// general scale (amax / MAX) would save up to one bit of int8's range (none of
// e4m3's) but let each of a page's up to page - 1 rescalings add half a step.
//
// HBM bound: the rows read once, one byte an element written.  One CTA per
// (page that gets rows, head, K or V); which pages those are is on the device,
// so the grid has a slot for each page that could: a sequence's rows from s to
// e touch at most e / page - s / page + 2 pages, so sequence i's slots start at
// row_start[i] / page + 2 i, which a CTA finds its sequence by.
#include "kv8.cuh"

namespace {

constexpr int kThreads = 128;
constexpr float kLeastScale = 7.8886090522101181e-31f;  // 2^-100

template <int FORMAT>
__device__ __forceinline__ float scale_for(float amax) {
    // amax = m 2^e, 1 <= m < 2; MAX = 1.984375 * 2^6 or 1.75 * 2^8
    const uint32_t bits = __float_as_uint(amax);
    const int top = FORMAT == kv8::kInt8 ? 6 : 8;
    const uint32_t most = FORMAT == kv8::kInt8 ? 0x7e0000u : 0x600000u;
    const int e = (int)(bits >> 23) - top + ((bits & 0x7fffffu) > most ? 1 : 0);
    return e < 27 ? kLeastScale : __uint_as_float((uint32_t)e << 23);
}

struct Args {
    kv8::Batch b;
    const void *k, *v;
    int64_t k_stride, v_stride;
    uint8_t *k_codes, *v_codes;
    float *k_scale, *v_scale;
    unsigned* status;
    int hkv, d;
};

template <typename T, int FORMAT>
__global__ void __launch_bounds__(kThreads) k_append(const __grid_constant__ Args a) {
    __shared__ float red[32];
    __shared__ int bad;
    const kv8::Batch& b = a.b;
    const int slot = blockIdx.x, head = blockIdx.y, page = 1 << b.page_shift;
    // the last sequence whose slots start at or before this one
    int lo = 0, hi = b.n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        const int start = min(max(b.row_start[mid], 0), b.rows);
        if ((start >> b.page_shift) + 2 * mid <= slot)
            lo = mid;
        else
            hi = mid - 1;
    }
    const kv8::Seq s = kv8::sequence(b, lo);
    const int first = max(s.first, 0);  // rows before position 0 are padding
    const int logical = (first >> b.page_shift) + slot - ((s.lo >> b.page_shift) + 2 * lo);
    const int64_t begin = (int64_t)logical << b.page_shift;
    if (s.n == 0 || logical < 0 || begin >= s.len) return;
    if (logical >= b.width) {
        if (threadIdx.x == 0) atomicOr(a.status, TB_B200_FLAG_POSITION_RANGE);
        return;
    }
    const int id = b.table[lo * b.table_stride + logical];
    if (id < 0 || id >= b.n_pages) {
        if (threadIdx.x == 0) atomicOr(a.status, TB_B200_FLAG_PAGE_RANGE);
        return;
    }
    const bool is_v = blockIdx.z != 0;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    const T* x = static_cast<const T*>(is_v ? a.v : a.k) + (int64_t)head * a.d;
    uint8_t* codes = (is_v ? a.v_codes : a.k_codes) +
                     (((int64_t)id * a.hkv + head) << b.page_shift) * a.d;
    float* scale = (is_v ? a.v_scale : a.k_scale) + (int64_t)id * a.hkv + head;
    // slots [from, to) of the page are new; slot from is row `row`
    const int from = max(first - (int)begin, 0);
    const int to = (int)min((int64_t)page, s.len - begin);
    const int row = s.lo + (int)(begin + from - s.first);
    const int n = (to - from) * a.d;
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();

    float amax = 0.0f;
    bool finite = true;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const float v = fabsf(tbk::Elt<T>::load(x + (row + i / a.d) * stride + i % a.d));
        if (v < INFINITY)
            amax = fmaxf(amax, v);
        else
            finite = false;
    }
    if (!finite) bad = 1;
    amax = tbk::block_max(amax, red);
    const float old = from > 0 ? *scale : 0.0f;
    const float now = fmaxf(scale_for<FORMAT>(amax), old);
    const float most = FORMAT == kv8::kInt8 ? 127.0f : 448.0f;
    if (now > old && from > 0) {
        const float ratio = old / now;
        for (int i = threadIdx.x; i < from * a.d; i += kThreads)
            codes[i] = kv8::encode<FORMAT>(kv8::decode<FORMAT>(codes[i]) * ratio);
    }
    const float per = 1.0f / now;  // both powers of two: exact
    for (int i = threadIdx.x; i < n; i += kThreads) {
        float v = tbk::Elt<T>::load(x + (row + i / a.d) * stride + i % a.d) * per;
        v = v != v ? 0.0f : fminf(fmaxf(v, -most), most);
        codes[from * a.d + i] = kv8::encode<FORMAT>(v);
    }
    __syncthreads();  // every thread has read *scale
    if (threadIdx.x == 0) {
        *scale = now;
        if (bad) atomicOr(a.status, TB_B200_FLAG_NONFINITE);
    }
}

}  // namespace

extern "C" int tb_b200_kv8_append(const TbB200Kv8* cache, const TbB200Kv8Batch* batch, int dtype,
                                  const void* k, int64_t k_stride, const void* v,
                                  int64_t v_stride, void* stream) {
    int rc = kv8::check_cache(cache, true);
    if (rc == TB_OK) rc = kv8::check_batch(batch, true);
    if (rc != TB_OK) return rc;
    if (dtype != TB_DTYPE_F32 && dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    const int64_t width = (int64_t)cache->n_kv_heads * cache->head_dim;
    if (batch->rows > 1 && (k_stride < width || v_stride < width)) return TB_ERR_INVALID_SHAPE;
    if (batch->rows == 0 || batch->n_seqs == 0) return TB_OK;
    if (!k || !v) return TB_ERR_INVALID_ARG;
    tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    const Args a = {kv8::view(cache, batch), k, v, k_stride, v_stride,
                    static_cast<uint8_t*>(cache->k), static_cast<uint8_t*>(cache->v),
                    cache->k_scale, cache->v_scale, ds->status, cache->n_kv_heads,
                    cache->head_dim};
    const dim3 grid((unsigned)(batch->rows / cache->page + 2 * batch->n_seqs),
                    (unsigned)cache->n_kv_heads, 2);
    cudaStream_t s = tbh::stream_of(stream);
    const bool f32 = dtype == TB_DTYPE_F32, int8 = cache->format == kv8::kInt8;
    if (f32 && int8)
        k_append<float, kv8::kInt8><<<grid, kThreads, 0, s>>>(a);
    else if (f32)
        k_append<float, kv8::kE4m3><<<grid, kThreads, 0, s>>>(a);
    else if (int8)
        k_append<__nv_bfloat16, kv8::kInt8><<<grid, kThreads, 0, s>>>(a);
    else
        k_append<__nv_bfloat16, kv8::kE4m3><<<grid, kThreads, 0, s>>>(a);
    TB_LAUNCH_CHECK("8-bit cache append kernel");
    return TB_OK;
}
