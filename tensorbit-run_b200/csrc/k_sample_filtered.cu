// k_sample_filtered.cu -- one token of each row of logits, after temperature, top-k, top-p
// and min-p.
//
//   w_i = exp((x_i - max x) / temperature) as a whole number of 2^-shift, shift = 62 - the
//   bits of the vocabulary, so that sums fit 64 bits and do not depend on an order;
//   the k first in falling order; of those the ones whose predecessors' weights sum to less
//   than top_p of all; of those the ones with w_i >= min_p; of those, in the order of i, the
//   first whose running sum is above u times the whole.
// A border in falling order is a pair (key, count): elements with a larger key are in, and of
// those with that key (a logit's bits in an order that compares like it) the first `count`.
// It is found digit by digit, 8 bits of the key at a time, from a histogram of the elements
// that share the digits found so far.
//
// A CTA a row, which is read from HBM once and from L2 after that.
#include <math.h>

#include "tb_device.cuh"
#include "tb_internal.h"

namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int64_t kMostVocab = 1 << 22;

struct Args {
    const void* logits;
    int64_t stride;
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    const double* uniforms;
    int32_t* out;
    int vocab, shift;
};

// Compares like the logit (-0 is 0); NaN is 0, below -infinity.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A row's weights.
struct Weights {
    float top;
    double temperature, unit;
    __device__ __forceinline__ double exact(float x) const {
        if (x == top) return 1.0;
        const double d = ((double)x - (double)top) / temperature;
        return d == d ? exp(d) : 0.0;  // NaN: a NaN, or (-infinity) / infinity
    }
    __device__ __forceinline__ unsigned long long operator()(float x) const {
        return __double2ull_rn(exact(x) * unit);
    }
};

struct Border {
    uint32_t key;
    int count;  // of the elements with that key
};

// floor(a b / 2^s), and whether anything was cut off.
__device__ __forceinline__ unsigned long long scaled(unsigned long long a, unsigned long long b,
                                                     int s, bool& cut) {
    const unsigned long long hi = __umul64hi(a, b), lo = a * b;
    cut = lo << (64 - s) != 0;
    return hi << (64 - s) | lo >> s;
}

struct Shared {
    unsigned int count[256];
    unsigned long long weight[256];
    unsigned long long warp_sum[kWarps];
    int warp_count[kWarps];
    float red[kWarps];
    uint32_t key;
    int chosen;
    unsigned long long before;
};

__device__ unsigned long long block_sum(unsigned long long v, Shared& sh) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(tbk::kFull, v, o);
    if ((threadIdx.x & 31) == 0) sh.warp_sum[threadIdx.x >> 5] = v;
    __syncthreads();
    unsigned long long s = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) s += sh.warp_sum[i];
    __syncthreads();
    return s;
}

// The border of the elements inside `in` (in falling order) where the sum of measure (1, or
// the weight) over the elements before one reaches `limit` > 0: the last element whose
// predecessors sum to less than limit.
template <typename T, bool BY_WEIGHT>
__device__ Border border_of(const T* x, const Args& a, const Weights& w, Border in,
                            unsigned long long limit, Shared& sh) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < 256; i += kThreads) {
            sh.count[i] = 0;
            sh.weight[i] = 0;
        }
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
            const float v = tbk::Elt<T>::load(x + i);
            const uint32_t k = key_of(v);
            if (k == 0 || (k & mask) != prefix || k < in.key) continue;
            atomicAdd(&sh.count[k >> shift & 255], 1u);
            if (BY_WEIGHT) atomicAdd(&sh.weight[k >> shift & 255], w(v));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long before = 0;  // relative to the digits before
            int d = 255, last = -1;
            unsigned long long last_before = 0;
            for (; d >= 0; --d) {
                if (sh.count[d] == 0) continue;
                if (before >= limit) break;
                last = d;
                last_before = before;
                unsigned long long here = BY_WEIGHT ? sh.weight[d] : sh.count[d];
                // a key at the outer border has only some of its elements inside
                if (shift == 0 && (prefix | d) == in.key)
                    here = BY_WEIGHT ? w(logit_of(in.key)) * in.count : in.count;
                before += here;
            }
            sh.chosen = max(last, 0);
            sh.before = last_before;
        }
        __syncthreads();
        prefix |= (uint32_t)sh.chosen << shift;
        limit -= sh.before;
        __syncthreads();
    }
    // of the elements with this key the ones whose predecessors sum to less than limit
    const unsigned long long each = BY_WEIGHT ? w(logit_of(prefix)) : 1ull;
    const int all = prefix == in.key ? in.count : (int)sh.count[prefix & 255];
    const unsigned long long n = each ? (limit + each - 1) / each : (unsigned long long)all;
    __syncthreads();
    return {prefix, (int)min((unsigned long long)all, n)};
}

template <typename T>
__global__ void __launch_bounds__(kThreads) k_sample(const Args a) {
    __shared__ Shared sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.stride;
    const int n = a.vocab;

    // the largest logit
    uint32_t top = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) top = max(top, key_of(tbk::Elt<T>::load(x + i)));
    top = __reduce_max_sync(tbk::kFull, top);
    if (lane == 0) sh.warp_count[warp] = (int)top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = max(top, (uint32_t)sh.warp_count[i]);
    __syncthreads();
    if (top <= key_of(-INFINITY)) {
        if (threadIdx.x == 0) a.out[row] = 0;
        return;
    }
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const float min_p = a.min_p ? a.min_p[row] : 0.0f;
    const bool greedy = !(t > 0.0f) || min_p > 1.0f;  // the first of the largest alone
    const Weights w = {logit_of(top), t > 0.0f ? (double)t : 1.0, (double)(1ull << a.shift)};

    // the elements inside: everything above -infinity at first
    Border in = {key_of(-INFINITY), 0};
    if (greedy) in = {top, 1};
    const int k = a.top_k ? a.top_k[row] : 0;
    if (!greedy && k > 0 && k < n) in = border_of<T, false>(x, a, w, in, k, sh);
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (!greedy && p < 1.0f) {
        unsigned long long sum = 0;
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const float v = tbk::Elt<T>::load(x + i);
            if (key_of(v) > in.key) sum += w(v);
        }
        sum = block_sum(sum, sh);
        sum += w(logit_of(in.key)) * in.count;
        bool cut;
        const unsigned long long q = p > 0.0f ? __double2ull_rd((double)p * 0x1p63) : 0ull;
        unsigned long long limit = scaled(sum, q, 63, cut);
        limit += cut;
        in = border_of<T, true>(x, a, w, in, max(limit, 1ull), sh);
    }
    const double least = min_p > 0.0f ? (double)min_p : 0.0;

    // warps' contiguous parts of the row, in order: elements with the border's key, then
    // weights inside
    const int per = (n + kWarps - 1) / kWarps, lo = min(n, warp * per), hi = min(n, lo + per);
    int ties = 0;
    for (int i = lo + lane; i < hi; i += 32) ties += key_of(tbk::Elt<T>::load(x + i)) == in.key;
    ties = __reduce_add_sync(tbk::kFull, ties);
    if (lane == 0) sh.warp_count[warp] = ties;
    __syncthreads();
    int tie0 = 0;
    for (int i = 0; i < warp; ++i) tie0 += sh.warp_count[i];
    auto inside = [&](int i, float v, int& seen) {  // a warp's 32 elements, in order
        const uint32_t key = i < hi ? key_of(v) : 0u;
        const uint32_t tied = __ballot_sync(tbk::kFull, key == in.key);
        const bool first = seen + __popc(tied & ((1u << lane) - 1)) < in.count;
        seen += __popc(tied);
        const bool is = key > in.key || (key == in.key && first);
        return is && (v == w.top || w.exact(v) >= least);
    };
    unsigned long long sum = 0;
    int seen = tie0;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const float v = i0 + lane < hi ? tbk::Elt<T>::load(x + i0 + lane) : 0.0f;
        if (inside(i0 + lane, v, seen)) sum += w(v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(tbk::kFull, sum, o);
    if (lane == 0) sh.warp_sum[warp] = sum;
    __syncthreads();
    unsigned long long all = 0, before = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        if (i < warp) before += sh.warp_sum[i];
        all += sh.warp_sum[i];
    }
    // the first with a running sum above u * all
    const double u = greedy ? 0.0 : a.uniforms[row];
    const unsigned long long uq =
        u > 0.0 ? min(__double2ull_rd(u * 0x1p53), (1ull << 53) - 1) : 0ull;
    bool cut;
    const unsigned long long target = scaled(all, uq, 53, cut);
    if (target < before || target >= before + sum) return;
    seen = tie0;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const float v = i0 + lane < hi ? tbk::Elt<T>::load(x + i0 + lane) : 0.0f;
        const unsigned long long mine = inside(i0 + lane, v, seen) ? w(v) : 0ull;
        unsigned long long run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long up = __shfl_up_sync(tbk::kFull, run, o);
            if (lane >= o) run += up;
        }
        const uint32_t past = __ballot_sync(tbk::kFull, before + run > target);
        if (past) {
            if (lane == 0) a.out[row] = i0 + __ffs(past) - 1;
            return;
        }
        before += __shfl_sync(tbk::kFull, run, 31);
    }
}

}  // namespace

extern "C" int tb_b200_sample(const TbB200Sample* t, void* stream) {
    if (!t) return TB_ERR_INVALID_ARG;
    if (t->dtype != TB_DTYPE_F32 && t->dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    if (t->rows < 0 || t->rows > INT32_MAX || t->vocab < 1 || t->vocab > kMostVocab ||
        (t->rows > 1 && t->stride < t->vocab))
        return TB_ERR_INVALID_SHAPE;
    if (t->rows == 0) return TB_OK;
    if (!t->logits || !t->uniforms || !t->out) return TB_ERR_INVALID_ARG;
    Args a = {t->logits, t->stride, t->temperature, t->top_p, t->min_p, t->top_k,
              t->uniforms, t->out, (int)t->vocab, 62};
    while ((1ll << (62 - a.shift)) < t->vocab) --a.shift;
    cudaStream_t s = tbh::stream_of(stream);
    if (t->dtype == TB_DTYPE_F32)
        k_sample<float><<<(unsigned)t->rows, kThreads, 0, s>>>(a);
    else
        k_sample<__nv_bfloat16><<<(unsigned)t->rows, kThreads, 0, s>>>(a);
    TB_LAUNCH_CHECK("filtered sampling kernel");
    return TB_OK;
}
