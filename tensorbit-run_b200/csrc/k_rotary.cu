// k_rotary.cu -- rotary positions of Q and K rows in both pair layouts, over
// part of the head or all of it, with an optional RMSNorm of each head in the
// same pass; and the frequencies, scaled for long contexts.
//
// Per row at position p, per pair i < r/2 of a head (r = rotary_dim):
//   a = p f_i,  (x0, x1) -> m (x0 cos a - x1 sin a, x1 cos a + x0 sin a)
// with (x0, x1) = (x[2i], x[2i+1]) or (x[i], x[i + r/2]), after
//   x -> x / sqrt(mean(x^2) + eps) * w
// over the whole head when the norm is asked for.
//
// The angle: an f32 product p f_i is off by 2^-24 p f_i, a hundredth of a
// turn at p = 10^6.  It is taken in double as turns, t = p (f_i / 2 pi), and
// t - rint(t), exact, goes to sincospif as an f32 and the remainder of that
// rounding by the first-order terms, so cos and sin carry the error of
// sincospif alone at every position.  r/2 such angles per row against
// (hq + hkv) d elements: under 1 % of the row's time.
//
// HBM bound: 2 (hq + hkv) d s bytes per row.  One CTA per row, so that a
// row's angles are computed once and shared; a group of G lanes owns a head,
// each lane two vectors of it that hold both elements of its pairs, so a
// head's sum of squares is a shuffle among G lanes and every element is read
// and written once, in place if asked.  A lane asks for the vectors of its
// first U heads before the angles are computed and keeps its pairs' cos and sin
// in registers for all of them; the CTA has just the threads that make its passes
// over the heads full ones.
//
// Measured: 16384 rows of 64 + 8 heads of 128, bf16, 94 us, 6.4 TB/s (a copy:
// 6.5; the first version, a head at a time: 127 us); norm and half the head, 4095
// rows of 32 + 32 heads of 128, f32, 46.1 us, 5.8 TB/s (49.6 with a division and a
// root rounded to nearest in rsqrtf's place); 777 rows of 32 + 32 heads of 80, f32,
// 8.4 us and 256 rows of 32 + 32 heads of 128, bf16, 5.5 us, where a launch and one
// row's chain of loads are most of the time.
#include <math.h>

#include "tb_device.cuh"
#include "tb_internal.h"

namespace {

using tbk::kFull;

constexpr int kMaxDim = 512;
constexpr int kThreads = 256;

// Most threads of a CTA.  The rotation of many rows alone streams best in small ones,
// that of few in large ones, of which four for every SM run at once: rows of 72 heads of
// 128 in bf16 with 128 and with 256 threads, 64 rows 3.4 and 3.0 us, 300 5.8 and 5.2, 592
// 7.4 and 6.9, 1024 9.5 and 10.2, 4096 27.4 and 29.0, 16384 94 and 101; of 9 heads of 256,
// 592 3.2 and 3.3, 1024 4.6 and 5.6, 8192 18 and 24.  With the norm, 592 9.4 and 8.5, 4095
// of f32 46.8 and 46.1 (but 1024 of bf16 12.1 and 13.4).
unsigned threads_of(bool norm, unsigned rows, int sm_count) {
    return norm || rows <= 4u * sm_count ? 256 : 128;
}

// ---------------------------------------------------------------- vectors
template <typename T, int VEC>
struct Vec {  // VEC = 1
    T e;
    __device__ static Vec load(const T* p) { return {*p}; }
    __device__ static Vec load_kept(const T* p) { return {*p}; }
    __device__ void widen(float (&v)[VEC]) const { v[0] = tbk::Elt<T>::load(&e); }
    __device__ static void store(T* p, const float (&v)[VEC]) { tbk::Elt<T>::store(p, v[0]); }
};

template <>
struct Vec<float, 4> {
    uint4 w;
    __device__ static Vec load(const float* p) { return {__ldcs(reinterpret_cast<const uint4*>(p))}; }
    __device__ static Vec load_kept(const float* p) { return {*reinterpret_cast<const uint4*>(p)}; }
    __device__ void widen(float (&v)[4]) const { tbk::Elt<float>::widen<4>(w, v); }
    __device__ static void store(float* p, const float (&v)[4]) { tbk::store_vec<float, 4>(p, v); }
};

template <>
struct Vec<__nv_bfloat16, 8> {
    uint4 w;
    __device__ static Vec load(const __nv_bfloat16* p) {
        return {__ldcs(reinterpret_cast<const uint4*>(p))};
    }
    __device__ static Vec load_kept(const __nv_bfloat16* p) {
        return {*reinterpret_cast<const uint4*>(p)};
    }
    __device__ void widen(float (&v)[8]) const { tbk::Elt<__nv_bfloat16>::widen<8>(w, v); }
    __device__ static void store(__nv_bfloat16* p, const float (&v)[8]) {
        tbk::store_vec<__nv_bfloat16, 8>(p, v);
    }
};

template <>
struct Vec<__nv_bfloat16, 4> {
    uint2 w;
    __device__ static Vec load(const __nv_bfloat16* p) {
        return {__ldcs(reinterpret_cast<const uint2*>(p))};
    }
    __device__ static Vec load_kept(const __nv_bfloat16* p) {
        return {*reinterpret_cast<const uint2*>(p)};
    }
    __device__ void widen(float (&v)[4]) const {
        v[0] = __uint_as_float(w.x << 16);
        v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16);
        v[3] = __uint_as_float(w.y & 0xffff0000u);
    }
    __device__ static void store(__nv_bfloat16* p, const float (&v)[4]) {
        *reinterpret_cast<uint2*>(p) =
            make_uint2(tbk::pack_bf16x2(v[0], v[1]), tbk::pack_bf16x2(v[2], v[3]));
    }
};

// ----------------------------------------------------------------- kernel
struct Args {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_stride, k_stride, q_out_stride, k_out_stride;
    const int32_t* positions;
    const double* freqs;
    const void *q_weight, *k_weight;
    float scale, eps, per;  // per: 1 / d
    int hq, hkv, d, r, group;
};

// scale * (cos, sin) of 2 pi t.
__device__ __forceinline__ float2 turn(double t, float scale) {
    const double part = t - rint(t);  // [-1/2, 1/2], exact
    const float x = (float)(2.0 * part);
    const float rest = (float)((2.0 * part - (double)x) * 3.14159265358979323846);
    float s, c;
    sincospif(x, &s, &c);
    return make_float2(scale * fmaf(-s, rest, c), scale * fmaf(c, rest, s));
}

template <typename T, int VEC, int NU, bool HALF, bool NORM>
__global__ void __launch_bounds__(kThreads, NU == 1 ? 4 : 1) k_rotary(const __grid_constant__ Args a) {
    __shared__ float2 cs[kMaxDim / 2];
    using V = Vec<T, VEC>;
    constexpr int U = NU == 1 ? 2 : 1;  // heads a lane holds at once
    const int64_t row = blockIdx.x;
    const int half = a.r / 2;
    const int lane = threadIdx.x % a.group, slot = threadIdx.x / a.group;
    const int per_pass = blockDim.x / a.group, heads = a.hq + a.hkv;
    const int nv = a.d / VEC, units = (nv + 1) / 2, hv = HALF ? half / VEC : 0;
    const T* q = static_cast<const T*>(a.q) + row * a.q_stride;
    const T* k = static_cast<const T*>(a.k) + row * a.k_stride - (int64_t)a.hq * a.d;
    T* q_out = static_cast<T*>(a.q_out) + row * a.q_out_stride;
    T* k_out = static_cast<T*>(a.k_out) + row * a.k_out_stride - (int64_t)a.hq * a.d;

    int at[NU][2];  // the lane's vectors of a head, nv where there is none
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        const int u = lane + n * a.group;
        // pairs of halves; past them, and for pairs side by side, two vectors: next
        // to each other, or half the head apart so that lanes stay next to lanes
        const bool split = HALF ? u < hv : VEC > 1;
        at[n][0] = split ? u : 2 * u;
        at[n][1] = split ? u + (HALF ? hv : units) : 2 * u + 1;
#pragma unroll
        for (int b = 0; b < 2; ++b)
            if (u >= units || at[n][b] > nv) at[n][b] = nv;
    }
    V held[U][NU][2];
    auto ask = [&](int h, V (&v)[NU][2]) {
        const T* in = (h < a.hq ? q : k) + (int64_t)h * a.d;
#pragma unroll
        for (int n = 0; n < NU; ++n)
#pragma unroll
            for (int b = 0; b < 2; ++b)
                if (h < heads && at[n][b] < nv) v[n][b] = V::load(in + at[n][b] * VEC);
    };
#pragma unroll
    for (int u = 0; u < U; ++u) ask(slot + u * per_pass, held[u]);

    if (half) {
        const double p = (double)a.positions[row];
        for (int i = threadIdx.x; i < half; i += blockDim.x)
            cs[i] = turn(p * (a.freqs[i] * 0.15915494309189533577), a.scale);
    }
    __syncthreads();
    // cos and sin of the lane's pairs: VEC of them, of (e, e) of the two vectors or
    // of (2 e, 2 e + 1) of the first, then the second; turns: whether they are pairs
    constexpr bool kAcross = HALF || VEC == 1;
    float2 t[NU][VEC];
    bool turns[NU][2];
#pragma unroll
    for (int n = 0; n < NU; ++n) {
        const int u = lane + n * a.group;
#pragma unroll
        for (int b = 0; b < 2; ++b)
            turns[n][b] = kAcross ? u < (HALF ? hv : half) : at[n][b] * VEC < a.r;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int b = kAcross ? 0 : 2 * e / VEC;
            const int i = kAcross ? u * VEC + e : at[n][b] * VEC / 2 + e % ((VEC + 1) / 2);
            if (turns[n][b]) t[n][e] = cs[i];
        }
    }

    for (int h0 = 0; h0 < heads; h0 += U * per_pass) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (h0 + u * per_pass >= heads) break;
            const int h = h0 + u * per_pass + slot;
            const bool is_q = h < a.hq, live = h < heads;
            T* out = (is_q ? q_out : k_out) + (int64_t)h * a.d;
            float x[NU][2][VEC];
            float ss = 0.0f;
#pragma unroll
            for (int n = 0; n < NU; ++n)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) x[n][b][e] = 0.0f;
                    if (live && at[n][b] < nv) held[u][n][b].widen(x[n][b]);
                    if (NORM) {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) ss = fmaf(x[n][b][e], x[n][b][e], ss);
                    }
                }
            if (NORM) {
                for (int o = a.group >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
                const float inv = rsqrtf(fmaf(ss, a.per, a.eps));  // 2 ulp
                const T* w = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
#pragma unroll
                for (int n = 0; n < NU; ++n)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        float g[VEC];
#pragma unroll
                        for (int e = 0; e < VEC; ++e) g[e] = 1.0f;
                        if (w && at[n][b] < nv) V::load_kept(w + at[n][b] * VEC).widen(g);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) x[n][b][e] = x[n][b][e] * inv * g[e];
                    }
            }
#pragma unroll
            for (int n = 0; n < NU; ++n) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if (!turns[n][kAcross ? 0 : 2 * e / VEC]) continue;
                    float& x0 = kAcross ? x[n][0][e] : x[n][2 * e / VEC][2 * e % VEC];
                    float& x1 = kAcross ? x[n][1][e] : x[n][2 * e / VEC][(2 * e + 1) % VEC];
                    const float y0 = x0 * t[n][e].x - x1 * t[n][e].y;
                    x1 = x1 * t[n][e].x + x0 * t[n][e].y;
                    x0 = y0;
                }
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    if (live && at[n][b] < nv) V::store(out + at[n][b] * VEC, x[n][b]);
            }
        }
        if (h0 + U * per_pass < heads) {
#pragma unroll
            for (int u = 0; u < U; ++u) ask(h0 + (U + u) * per_pass + slot, held[u]);
        }
    }
}

template <typename T, int VEC, int NU, bool NORM>
void launch_layout(const Args& a, bool half_layout, unsigned rows, int sm_count,
                   cudaStream_t s) {
    // the fewest passes over the heads, and the fewest threads for as many
    const int64_t lanes = (int64_t)(a.hq + a.hkv) * a.group;
    const unsigned most = threads_of(NORM, rows, sm_count);
    const int64_t passes = (lanes + most - 1) / most;
    const unsigned threads = (unsigned)((lanes + passes * 32 - 1) / (passes * 32) * 32);
    if (half_layout)
        k_rotary<T, VEC, NU, true, NORM><<<rows, threads, 0, s>>>(a);
    else
        k_rotary<T, VEC, NU, false, NORM><<<rows, threads, 0, s>>>(a);
}

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Whether every vector of VEC elements starts on its own size and no vector
// holds elements of two kinds (a pair's first and second half, rotated and not).
bool vectors_of(int vec, size_t s, const Args& a, bool half_layout) {
    const size_t bytes = vec * s;
    return a.d % vec == 0 && (half_layout ? a.r / 2 : a.r) % vec == 0 &&
           (!a.hq || (aligned(a.q, bytes) && aligned(a.q_out, bytes) && a.q_stride % vec == 0 &&
                      a.q_out_stride % vec == 0)) &&
           (!a.hkv || (aligned(a.k, bytes) && aligned(a.k_out, bytes) && a.k_stride % vec == 0 &&
                       a.k_out_stride % vec == 0)) &&
           aligned(a.q_weight, bytes) && aligned(a.k_weight, bytes);
}

// Lanes per head: a power of two that covers the head's units, 32 at most.
int group_of(int d, int vec) {
    const int units = (d / vec + 1) / 2;
    int g = 1;
    while (g < units && g < 32) g <<= 1;
    return g;
}

template <bool NORM>
void launch(Args& a, int dtype, bool half_layout, unsigned rows, int sm_count, cudaStream_t s) {
    if (dtype == TB_DTYPE_BF16) {
        if (vectors_of(8, 2, a, half_layout)) {
            a.group = group_of(a.d, 8);
            launch_layout<__nv_bfloat16, 8, 1, NORM>(a, half_layout, rows, sm_count, s);
        } else if (vectors_of(4, 2, a, half_layout)) {
            a.group = group_of(a.d, 4);
            if (a.d <= 256)
                launch_layout<__nv_bfloat16, 4, 1, NORM>(a, half_layout, rows, sm_count, s);
            else
                launch_layout<__nv_bfloat16, 4, 2, NORM>(a, half_layout, rows, sm_count, s);
        } else {
            a.group = 32;
            launch_layout<__nv_bfloat16, 1, 8, NORM>(a, half_layout, rows, sm_count, s);
        }
    } else if (vectors_of(4, 4, a, half_layout)) {
        a.group = group_of(a.d, 4);
        if (a.d <= 256)
            launch_layout<float, 4, 1, NORM>(a, half_layout, rows, sm_count, s);
        else
            launch_layout<float, 4, 2, NORM>(a, half_layout, rows, sm_count, s);
    } else {
        a.group = 32;
        launch_layout<float, 1, 8, NORM>(a, half_layout, rows, sm_count, s);
    }
}

int run(const TbB200Rotary* t, bool norm, void* stream) {
    if (!t) return TB_ERR_INVALID_ARG;
    if (t->rows < 0 || t->rows > INT32_MAX || t->n_q_heads < 0 || t->n_kv_heads < 0 ||
        (int64_t)t->n_q_heads + t->n_kv_heads > INT32_MAX / 2 ||  // heads of passes past it too
        t->head_dim < 1 || t->head_dim > kMaxDim || t->rotary_dim < 0 ||
        t->rotary_dim > t->head_dim || t->rotary_dim % 2)
        return TB_ERR_INVALID_SHAPE;
    if (t->dtype != TB_DTYPE_F32 && t->dtype != TB_DTYPE_BF16) return TB_ERR_UNSUPPORTED_DTYPE;
    if (t->layout != TB_B200_ROTARY_INTERLEAVED && t->layout != TB_B200_ROTARY_HALF)
        return TB_ERR_INVALID_ARG;
    const int64_t dq = (int64_t)t->n_q_heads * t->head_dim, dk = (int64_t)t->n_kv_heads * t->head_dim;
    if (t->rows > 1 && ((dq && (t->q_stride < dq || t->q_out_stride < dq)) ||
                        (dk && (t->k_stride < dk || t->k_out_stride < dk))))
        return TB_ERR_INVALID_SHAPE;
    if (t->rows == 0 || dq + dk == 0) return TB_OK;
    if ((dq && (!t->q || !t->q_out)) || (dk && (!t->k || !t->k_out)) ||
        (t->rotary_dim && (!t->positions || !t->freqs)))
        return TB_ERR_INVALID_ARG;
    if ((dq && t->q == t->q_out && t->q_stride != t->q_out_stride && t->rows > 1) ||
        (dk && t->k == t->k_out && t->k_stride != t->k_out_stride && t->rows > 1))
        return TB_ERR_INVALID_ARG;
    Args a = {t->q,         t->k,     t->q_out,    t->k_out,    t->q_stride,    t->k_stride,
              t->q_out_stride, t->k_out_stride, t->positions, t->freqs,
              norm ? t->q_weight : nullptr, norm ? t->k_weight : nullptr, t->scale, t->eps,
              1.0f / (float)t->head_dim,
              t->n_q_heads, t->n_kv_heads, t->head_dim, t->rotary_dim, 0};
    const tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    cudaStream_t s = tbh::stream_of(stream);
    const bool half_layout = t->layout == TB_B200_ROTARY_HALF;
    if (norm)
        launch<true>(a, t->dtype, half_layout, (unsigned)t->rows, ds->sm_count, s);
    else
        launch<false>(a, t->dtype, half_layout, (unsigned)t->rows, ds->sm_count, s);
    TB_LAUNCH_CHECK("rotary kernel");
    return TB_OK;
}

// ------------------------------------------------------------ frequencies
// One block, a thread per pair; pow in double (f_i spans five decades, and an
// error of 2^-24 in it is one of 2^-24 p f_i in the angle).
__global__ void __launch_bounds__(kMaxDim / 2)
k_rotary_freqs(int kind, int r, double theta, double factor, double trained, double low,
               double high, double* freqs) {
    const int i = threadIdx.x;
    if (i >= r / 2) return;
    double f = pow(theta, -2.0 * i / r);
    if (kind == TB_B200_ROTARY_SCALE_LINEAR) {
        f = f / factor;
    } else if (kind == TB_B200_ROTARY_SCALE_BANDS) {
        const double turns = trained * f / 6.283185307179586476925;
        const double keep = fmin(fmax((turns - low) / (high - low), 0.0), 1.0);
        f = f * ((1.0 - keep) / factor + keep);
    } else if (kind == TB_B200_ROTARY_SCALE_YARN) {  // low, high: first and last pair of the ramp
        const double width = high == low ? 0.001 : high - low;
        const double ramp = fmin(fmax((i - low) / width, 0.0), 1.0);
        f = f * (1.0 - ramp) + f / factor * ramp;
    }
    freqs[i] = f;
}

}  // namespace

extern "C" int tb_b200_rotary(const TbB200Rotary* rotary, void* stream) {
    return run(rotary, false, stream);
}

extern "C" int tb_b200_qk_norm_rotary(const TbB200Rotary* rotary, void* stream) {
    return run(rotary, true, stream);
}

extern "C" int tb_b200_rotary_freqs(int rotary_dim, const TbB200RotaryScaling* scaling,
                                    double* freqs_dev, void* stream) {
    if (!scaling || !freqs_dev) return TB_ERR_INVALID_ARG;
    if (rotary_dim < 2 || rotary_dim > kMaxDim || rotary_dim % 2) return TB_ERR_INVALID_SHAPE;
    const int r = rotary_dim;
    double theta = scaling->theta, low = scaling->low, high = scaling->high;
    const bool banded = scaling->kind == TB_B200_ROTARY_SCALE_BANDS ||
                        scaling->kind == TB_B200_ROTARY_SCALE_YARN;
    if (scaling->kind < TB_B200_ROTARY_SCALE_NONE || scaling->kind > TB_B200_ROTARY_SCALE_YARN ||
        !(theta > 0.0) || !isfinite(theta))
        return TB_ERR_INVALID_ARG;
    if (scaling->kind != TB_B200_ROTARY_SCALE_NONE &&
        (!(scaling->factor > 0.0) || !isfinite(scaling->factor)))
        return TB_ERR_INVALID_ARG;
    if (banded && (!(scaling->trained > 0.0) || !isfinite(scaling->trained) || !(low > 0.0) ||
                   !(high > low) || !isfinite(high)))
        return TB_ERR_INVALID_ARG;
    if (scaling->kind == TB_B200_ROTARY_SCALE_NTK) {
        if (r == 2) return TB_ERR_INVALID_SHAPE;
        theta *= pow(scaling->factor, (double)r / (r - 2));
    } else if (scaling->kind == TB_B200_ROTARY_SCALE_YARN) {
        if (theta == 1.0) return TB_ERR_INVALID_ARG;
        const double per = r / (2.0 * log(theta)), whole = scaling->trained / (2.0 * M_PI);
        const double first = fmax(floor(per * log(whole / high)), 0.0);
        const double last = fmin(ceil(per * log(whole / low)), r - 1.0);
        low = first;
        high = last;
    }
    k_rotary_freqs<<<1, kMaxDim / 2, 0, tbh::stream_of(stream)>>>(
        scaling->kind, r, theta, scaling->factor, scaling->trained, low, high, freqs_dev);
    TB_LAUNCH_CHECK("rotary frequencies kernel");
    return TB_OK;
}
