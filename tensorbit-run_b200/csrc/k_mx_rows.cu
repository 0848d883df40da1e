// k_mx_rows.cu -- rows to microscaled formats (mx.cuh): quantised as they are, behind
// SwiGLU, or behind a residual add and RMSNorm; and back to values.
//
// A thread has 32 bytes of a row (16 where rows are reduced first: the norm), so a block of 32
// elements is 2 to 8 neighbouring lanes, its largest magnitude 1 to 3 shuffles, and the four
// scales of a tile's row one 32-bit store.  Bytes are the inputs once, codes and scales once;
// what bounds the kernels now is their instructions (issue slots are 75 % busy, DRAM 41 to
// 51 %), most of which widen, scale and round:
//   28672 x 8192 bf16 to 4 bits 230 us (5.1 TB/s); 283 with 16 bytes a thread, more with two
//   or four pieces of work a thread
//   SwiGLU 4096 x 28672 bf16 140 us (4.2 TB/s)
//   norm 16384 x 8192 bf16 with the residual 198 us (4.8 TB/s); 188 with products rounded twice
#include <cmath>

#include "bodies.cuh"
#include "mx.cuh"

namespace {

using tbk::Elt;

constexpr int kThreads = 256;

// W times 16 bytes of a row as they are.
template <typename T, int W>
struct Chunk {
    static constexpr int V = Elt<T>::kVec, E = W * V;
    uint4 r[W];

    // Elements [at, at + E) of a row of `cols`, zeros past its end; vec: 16-byte aligned.
    __device__ __forceinline__ void load(const T* row, int at, int cols, bool vec) {
        if (vec && at + E <= cols) {
#pragma unroll
            for (int j = 0; j < W; ++j) r[j] = __ldcs(reinterpret_cast<const uint4*>(row + at) + j);
            return;
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[i] = 0;
                if constexpr (sizeof(T) == 4) {
                    const int k = at + j * V + i;
                    if (k < cols) w[i] = reinterpret_cast<const uint32_t*>(row)[k];
                } else {
                    const uint16_t* u = reinterpret_cast<const uint16_t*>(row);
                    const int k = at + j * V + 2 * i;
                    if (k < cols) w[i] = u[k];
                    if (k + 1 < cols) w[i] |= (uint32_t)u[k + 1] << 16;
                }
            }
            r[j] = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    __device__ __forceinline__ void widen(float (&v)[E]) const {
#pragma unroll
        for (int j = 0; j < W; ++j) {
            float part[V];
            Elt<T>::template widen<V>(r[j], part);
#pragma unroll
            for (int i = 0; i < V; ++i) v[j * V + i] = part[i];
        }
    }
};

// Elements [at, at + E) of a row of `cols` from v.
template <typename T, int E>
__device__ __forceinline__ void store_chunk(T* row, int at, int cols, bool vec,
                                            const float (&v)[E]) {
    if (vec && at + E <= cols) {
        constexpr int V = Elt<T>::kVec;
#pragma unroll
        for (int i = 0; i < E; i += V) {
            float part[V];
#pragma unroll
            for (int j = 0; j < V; ++j) part[j] = v[i + j];
            tbk::store_vec<T, V>(row + at + i, part);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (at + i < cols) Elt<T>::store(row + at + i, v[i]);
}

// Row and chunk of an item; 32-bit division where the items fit.
__device__ __forceinline__ void place_of(int64_t i, int chunks, bool small, int64_t& r, int& c) {
    if (small) {
        const uint32_t q = (uint32_t)i / (uint32_t)chunks;
        r = q;
        c = (int)((uint32_t)i - q * (uint32_t)chunks);
    } else {
        r = i / chunks;
        c = (int)(i - r * chunks);
    }
}

// ------------------------------------------------- quantise, SwiGLU
template <typename T>
struct Rows {
    const T *a, *b;  // b: SwiGLU's up rows, a its gate rows
    int64_t a_stride, b_stride;
    bool vec;
};

// tbk::silu_f of E elements, the same bits with a shorter division: q = g r, r an approximate
// reciprocal of d = 1 + e^-g after one of Newton's steps, and q + r (g - q d) is the quotient
// rounded to nearest (Markstein's theorems) where nothing leaves f32's normal numbers and d's
// mantissa is not all ones, r then being the nearest to 1 / d.  With all ones r may be 2^-k in
// place of 2^-k (1 + 2^-23), and the quotient comes out wrong only for g = 2^j: of those, 2^-23
// alone has such a d.  (Compared for every f32.  4096 rows of 28672 in bf16: 153 us with the exact
// division's own checks, 140 so.)
template <int E>
__device__ __forceinline__ void silu(float (&v)[E]) {
    float most = 0.0f, least = INFINITY;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
        const float x = fabsf(v[i]), y = fabsf(v[i + 1]);
        asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(most) : "f"(most), "f"(x), "f"(y));
        asm("min.f32 %0, %1, %2, %3;" : "=f"(least) : "f"(least), "f"(x), "f"(y));
    }
    if (!(most < 80.0f) || least < 0x1p-22f) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = tbk::silu_f(v[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float d = __fadd_rn(1.0f, expf(-v[i]));
        float r;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
        r = fmaf(r, fmaf(-d, r, 1.0f), r);
        const float q = v[i] * r;
        v[i] = fmaf(r, fmaf(-q, d, v[i]), q);
    }
}

// A thread an item: chunk c of row r, all rows of whole tiles (behind the last one only the
// scales are written).
template <typename T, int FORMAT, bool SWIGLU>
__global__ void __launch_bounds__(kThreads) k_rows(const Rows<T> in, const mx::View out,
                                                   int chunks, int64_t items, bool small) {
    using C = Chunk<T, 2>;
    constexpr int E = C::E;
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    int64_t r;
    int c;
    place_of(min(i, items - 1), chunks, small, r, c);
    const bool live = i < items && r < out.rows;
    C x, y;
    if (live) {
        x.load(in.a + r * in.a_stride, c * E, out.cols, in.vec);
        if constexpr (SWIGLU) y.load(in.b + r * in.b_stride, c * E, out.cols, in.vec);
    } else {
        x.r[0] = x.r[1] = y.r[0] = y.r[1] = make_uint4(0, 0, 0, 0);
    }
    float v[E];
    x.widen(v);
    if constexpr (SWIGLU) {
        float u[E];
        y.widen(u);
        silu<E>(v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = __fmul_rn(v[e], u[e]);
    }
    mx::store_block<FORMAT, E>(out, r, c, live, v);
    if (!live && i < items && c % (128 / E) == 0)
        *reinterpret_cast<uint32_t*>(out.scales + mx::scales_at(r, c * E / 128, out.tiles)) = 0;
}

template <typename T, bool SWIGLU>
int launch_rows(const Rows<T>& in, const TbB200Mx* out, cudaStream_t s) {
    const mx::View v = mx::view(out);
    const int chunks = v.tiles * (128 / Chunk<T, 2>::E);
    const int64_t items = mx::tiles_of(v.rows) * 128 * chunks;
    const int64_t grid = (items + kThreads - 1) / kThreads;
    if (grid > INT32_MAX) return TB_ERR_INVALID_SHAPE;
    const bool small = items + kThreads <= UINT32_MAX;
    if (out->format == mx::kE4m3)
        k_rows<T, mx::kE4m3, SWIGLU><<<(unsigned)grid, kThreads, 0, s>>>(in, v, chunks, items, small);
    else
        k_rows<T, mx::kE2m1, SWIGLU><<<(unsigned)grid, kThreads, 0, s>>>(in, v, chunks, items, small);
    TB_LAUNCH_CHECK("microscaled rows kernel");
    return TB_OK;
}

template <typename T>
bool aligned_rows(const void* p, int64_t stride) {
    return tbh::aligned16(p) && stride * (int64_t)sizeof(T) % 16 == 0;
}

template <typename T>
int quantize(const void* x, int64_t stride, const TbB200Mx* out, cudaStream_t s) {
    const Rows<T> in = {static_cast<const T*>(x), nullptr, stride, 0, aligned_rows<T>(x, stride)};
    return launch_rows<T, false>(in, out, s);
}

template <typename T>
int swiglu(const void* gate, int64_t gate_stride, const void* up, int64_t up_stride,
           const TbB200Mx* out, cudaStream_t s) {
    const Rows<T> in = {static_cast<const T*>(gate), static_cast<const T*>(up), gate_stride,
                        up_stride,
                        aligned_rows<T>(gate, gate_stride) && aligned_rows<T>(up, up_stride)};
    return launch_rows<T, true>(in, out, s);
}

// ------------------------------------------------- back to values
// A thread 16 codes.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(kThreads) k_values(const mx::View t, T* y, int64_t stride,
                                                     bool vec, int chunks, int64_t items,
                                                     bool small) {
    const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (i >= items) return;
    int64_t r;
    int c;
    place_of(i, chunks, small, r, c);
    const uint8_t* from = t.codes + r * t.pitch + (int64_t)c * (FORMAT == mx::kE4m3 ? 16 : 8);
    const float scale = mx::value_of(t.scales[mx::scales_at(r, c / 8, t.tiles) + c / 2 % 4]);
    float v[16];
    if constexpr (FORMAT == mx::kE4m3) {
        const uint4 w = *reinterpret_cast<const uint4*>(from);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint16_t two = (uint16_t)((&w.x)[j / 2] >> j % 2 * 16);
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(two, __NV_E4M3);
            v[2 * j] = __half2float(__half(__half_raw{h.x}));
            v[2 * j + 1] = __half2float(__half(__half_raw{h.y}));
        }
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(from);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            // sign, 2 exponent bits and 1 mantissa bit sit in f32's places 126 binades of
            // bias below their value, the subnormal 0.5 included
            const uint32_t n = (j < 8 ? w.x : w.y) >> j % 8 * 4;
            v[j] = __uint_as_float((n & 8) << 28 | (n & 7) << 22) * 8.5070591730234616e37f;
        }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] *= scale;
    store_chunk<T, 16>(y + r * stride, c * 16, t.cols, vec, v);
}

template <typename T>
int dequantize(const TbB200Mx* t, void* y, int64_t stride, cudaStream_t s) {
    const mx::View v = mx::view(t);
    const int chunks = (v.cols + 15) / 16;
    const int64_t items = v.rows * chunks, grid = (items + kThreads - 1) / kThreads;
    if (grid > INT32_MAX) return TB_ERR_INVALID_SHAPE;
    const bool vec = aligned_rows<T>(y, stride), small = items + kThreads <= UINT32_MAX;
    if (t->format == mx::kE4m3)
        k_values<T, mx::kE4m3><<<(unsigned)grid, kThreads, 0, s>>>(v, static_cast<T*>(y), stride,
                                                                   vec, chunks, items, small);
    else
        k_values<T, mx::kE2m1><<<(unsigned)grid, kThreads, 0, s>>>(v, static_cast<T*>(y), stride,
                                                                   vec, chunks, items, small);
    TB_LAUNCH_CHECK("microscaled values kernel");
    return TB_OK;
}

// ------------------------------------------------- residual + RMSNorm
template <typename T>
struct Norm {
    const T *x, *res, *w;
    T* h;
    bool vec, vec_w;
    float eps;
    double root;  // of the number of columns
};

// h of a chunk: x + residual in f32, the same bits each time.
template <typename T>
__device__ __forceinline__ void sum_of(const Norm<T>& in, const Chunk<T, 1>& x, const Chunk<T, 1>& res,
                                       float (&h)[Chunk<T, 1>::E]) {
    x.widen(h);
    if (in.res) {
        float r[Chunk<T, 1>::E];
        res.widen(r);
#pragma unroll
        for (int e = 0; e < Chunk<T, 1>::E; ++e) h[e] = __fadd_rn(h[e], r[e]);
    }
}

// The norm's factor: (hi + lo) by, by a power of two that keeps hi and its products with h
// within f32's normal numbers for rows of any size.
struct Factor {
    float hi, lo, by;
};

// The norm of chunk c of row r, stored; h comes scaled by the factor's power of two.
template <typename T, int FORMAT>
__device__ __forceinline__ void finish(const Norm<T>& in, const mx::View& out, int64_t r, int c,
                                       bool live, Factor scale, float (&h)[Chunk<T, 1>::E]) {
    constexpr int E = Chunk<T, 1>::E;
    // h times the factor's two parts times w, to half an ulp and a little: what a product's
    // rounding leaves out goes on with it (each step as it is written: a sum that took the last
    // product unrounded would count what that left out twice)
    float w[E];
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = 1.0f;
    if (in.w && live) {
        if (in.vec_w && c * E + E <= out.cols) {
            Chunk<T, 1> raw;
            raw.r[0] = *reinterpret_cast<const uint4*>(in.w + c * E);
            raw.widen(w);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                w[e] = c * E + e < out.cols ? Elt<T>::load(in.w + c * E + e) : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float t = __fmul_rn(h[e], scale.hi), y = __fmul_rn(t, w[e]);
        const float left = fmaf(h[e], scale.lo, fmaf(h[e], scale.hi, -t));
        h[e] = __fadd_rn(y, fmaf(left, w[e], fmaf(t, w[e], -y)));
    }
    if (c * E + E > out.cols) {  // (a row whose scale is NaN has fill of zeros all the same)
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (c * E + e >= out.cols) h[e] = 0.0f;
    }
    mx::store_block<FORMAT, E>(out, r, c, live, h);
}

// The norm's factor from the sum of squares, as two f32: an error of it moves a whole row's
// codes the same way, over the same rounding borders.
__device__ __forceinline__ Factor scale_of(double ss, float eps, double root) {
    const double s = rsqrt(ss + (double)eps) * root;  // off by less than 2^-51
    const bool great = s > 0x1p64, small = s < 0x1p-64;
    const float by = great ? 0x1p64f : small ? 0x1p-64f : 1.0f;
    const double rest = s * (great ? 0x1p-64 : small ? 0x1p64 : 1.0);
    const float hi = (float)rest;
    return {hi, hi < INFINITY ? (float)(rest - (double)hi) : 0.0f, by};
}
// The sum over a row's G threads (tbk::group_sum's), in double.
__device__ __forceinline__ double row_sum(double v, int G, double* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(tbk::kFull, v, o);
    if (G <= 32) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int first = threadIdx.x / G * (G >> 5);
    double s = red[first];
    for (int w = 1; w < (G >> 5); ++w) s += red[first + w];
    return s;
}
// The sum of a chunk's squares.  Double holds each exactly whatever the row's size; f32's overflow
// above 1.8e19 and vanish below 1e-23, and a narrow row's sum of them is off by more than the
// factor's second part says.  (16384 rows of 8192 bf16: 198 us with either.)
template <int E>
__device__ __forceinline__ double squares(const float (&h)[E]) {
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) sum = fma((double)h[e], (double)h[e], sum);
    return sum;
}

// G threads a row, ITEMS chunks a thread, whose sums stay in registers.
template <typename T, int FORMAT, int ITEMS, int MAXT>
__global__ void __launch_bounds__(MAXT) k_norm(const Norm<T> in, const mx::View out, int G) {
    constexpr int E = Chunk<T, 1>::E;
    __shared__ double red[32];
    const int lane = threadIdx.x & (G - 1);
    const int64_t r = (int64_t)blockIdx.x * (blockDim.x / G) + threadIdx.x / G;
    const bool active = r < out.rows;
    const int chunks = out.tiles * (128 / E);
    float h[ITEMS][E];
    double ss = 0.0;
    if (active) {
        Chunk<T, 1> x[ITEMS], res[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = lane + i * G;
            if (c < chunks) {
                x[i].load(in.x + r * out.cols, c * E, out.cols, in.vec);
                if (in.res) res[i].load(in.res + r * out.cols, c * E, out.cols, in.vec);
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (lane + i * G < chunks) {
                sum_of(in, x[i], res[i], h[i]);
                if (in.h)
                    store_chunk<T, E>(in.h + r * out.cols, (lane + i * G) * E, out.cols, in.vec, h[i]);
                ss += squares<E>(h[i]);
            }
        }
    }
    ss = row_sum(ss, G, red);
    const Factor scale = scale_of(ss, in.eps, in.root);
    if (scale.by != 1.0f) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) h[i][e] *= scale.by;
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        const int c = lane + i * G;
        const bool live = active && c < chunks;
        if (!live) {
#pragma unroll
            for (int e = 0; e < E; ++e) h[i][e] = 0.0f;
        }
        finish<T, FORMAT>(in, out, r, c, live, scale, h[i]);
        if (!active && c < chunks && r < (out.rows + 127) / 128 * 128 && c % (128 / E) == 0)
            *reinterpret_cast<uint32_t*>(out.scales + mx::scales_at(r, c * E / 128, out.tiles)) = 0;
    }
}

// Rows wider than that: a CTA a row, read twice, the second time from L2.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(1024) k_norm_wide(const Norm<T> in, const mx::View out) {
    constexpr int E = Chunk<T, 1>::E;
    __shared__ double red[32];
    const int64_t r = blockIdx.x;
    const int chunks = out.tiles * (128 / E);
    const bool active = r < out.rows;
    double ss = 0.0;
    Chunk<T, 1> x, res;
    float h[E];
    for (int c = threadIdx.x; active && c < chunks; c += blockDim.x) {
        x.load(in.x + r * out.cols, c * E, out.cols, in.vec);
        if (in.res) res.load(in.res + r * out.cols, c * E, out.cols, in.vec);
        sum_of(in, x, res, h);
        ss += squares<E>(h);
    }
    ss = row_sum(ss, blockDim.x, red);
    const Factor scale = scale_of(ss, in.eps, in.root);
    for (int c0 = 0; c0 < chunks; c0 += blockDim.x) {
        const int c = c0 + threadIdx.x;
        const bool live = active && c < chunks;
#pragma unroll
        for (int e = 0; e < E; ++e) h[e] = 0.0f;
        if (live) {
            x.load(in.x + r * out.cols, c * E, out.cols, in.vec);
            if (in.res) res.load(in.res + r * out.cols, c * E, out.cols, in.vec);
            sum_of(in, x, res, h);
            if (in.h) store_chunk<T, E>(in.h + r * out.cols, c * E, out.cols, in.vec, h);
#pragma unroll
            for (int e = 0; e < E; ++e) h[e] *= scale.by;
        }
        finish<T, FORMAT>(in, out, r, c, live, scale, h);
        if (!active && c < chunks && c % (128 / E) == 0)
            *reinterpret_cast<uint32_t*>(out.scales + mx::scales_at(r, c * E / 128, out.tiles)) = 0;
    }
}

template <typename T, int FORMAT>
int launch_norm(const Norm<T>& in, const TbB200Mx* y, cudaStream_t s) {
    const mx::View out = mx::view(y);
    const int64_t rows = mx::tiles_of(out.rows) * 128;
    const tbh::NormCfg c = tbh::norm_cfg((int64_t)out.tiles * (128 / Chunk<T, 1>::E), 1024);
    const int per = c.threads / c.G;
    const unsigned grid = (unsigned)((rows + per - 1) / per);
    if (c.items == 0) {
        k_norm_wide<T, FORMAT><<<(unsigned)rows, 1024, 0, s>>>(in, out);
    } else if (c.threads <= 256) {
        switch (c.items) {
            case 1: k_norm<T, FORMAT, 1, 256><<<grid, c.threads, 0, s>>>(in, out, c.G); break;
            case 2: k_norm<T, FORMAT, 2, 256><<<grid, c.threads, 0, s>>>(in, out, c.G); break;
            default: k_norm<T, FORMAT, 4, 256><<<grid, c.threads, 0, s>>>(in, out, c.G); break;
        }
    } else {
        switch (c.items) {
            case 1: k_norm<T, FORMAT, 1, 1024><<<grid, c.threads, 0, s>>>(in, out, c.G); break;
            case 2: k_norm<T, FORMAT, 2, 1024><<<grid, c.threads, 0, s>>>(in, out, c.G); break;
            default: k_norm<T, FORMAT, 4, 1024><<<grid, c.threads, 0, s>>>(in, out, c.G); break;
        }
    }
    TB_LAUNCH_CHECK("residual_rms_norm_mx kernel");
    return TB_OK;
}

template <typename T>
int norm(const void* x, const void* res, const void* w, void* h, const TbB200Mx* y, float eps,
         cudaStream_t s) {
    const bool vec = aligned_rows<T>(x, y->cols) && (!res || tbh::aligned16(res)) &&
                     (!h || tbh::aligned16(h));
    const Norm<T> in = {static_cast<const T*>(x), static_cast<const T*>(res),
                        static_cast<const T*>(w), static_cast<T*>(h), vec, tbh::aligned16(w), eps,
                        std::sqrt((double)y->cols)};
    return y->format == mx::kE4m3 ? launch_norm<T, mx::kE4m3>(in, y, s)
                                  : launch_norm<T, mx::kE2m1>(in, y, s);
}

bool is_float(int dtype) { return dtype == TB_DTYPE_F32 || dtype == TB_DTYPE_BF16; }

// Rows of cols elements that are `stride` apart.
bool strided(int64_t rows, int64_t cols, int64_t stride) { return rows <= 1 || stride >= cols; }

}  // namespace

extern "C" int tb_b200_mx_bytes(int format, int64_t rows, int64_t cols, size_t* codes,
                                size_t* scales) {
    const TbB200Mx t = {format, rows, cols, nullptr, nullptr};
    const int rc = mx::check(&t, false);
    if (rc != TB_OK) return rc;
    if (!codes || !scales) return TB_ERR_INVALID_ARG;
    *codes = (size_t)(rows * mx::pitch_of(format, cols));
    *scales = (size_t)(mx::tiles_of(rows) * mx::tiles_of(cols) * mx::kTileBytes);
    return TB_OK;
}

extern "C" int tb_b200_mx_quantize(int dtype, const void* x, int64_t x_stride,
                                   const TbB200Mx* out, void* stream) {
    const int rc = mx::check(out, true);
    if (rc != TB_OK) return rc;
    if (!is_float(dtype)) return TB_ERR_UNSUPPORTED_DTYPE;
    if (!strided(out->rows, out->cols, x_stride)) return TB_ERR_INVALID_SHAPE;
    if (out->rows == 0) return TB_OK;
    if (!x) return TB_ERR_INVALID_ARG;
    cudaStream_t s = tbh::stream_of(stream);
    return dtype == TB_DTYPE_F32 ? quantize<float>(x, x_stride, out, s)
                                 : quantize<__nv_bfloat16>(x, x_stride, out, s);
}

extern "C" int tb_b200_mx_dequantize(const TbB200Mx* t, int dtype, void* y, int64_t y_stride,
                                     void* stream) {
    const int rc = mx::check(t, true);
    if (rc != TB_OK) return rc;
    if (!is_float(dtype)) return TB_ERR_UNSUPPORTED_DTYPE;
    if (!strided(t->rows, t->cols, y_stride)) return TB_ERR_INVALID_SHAPE;
    if (t->rows == 0) return TB_OK;
    if (!y) return TB_ERR_INVALID_ARG;
    cudaStream_t s = tbh::stream_of(stream);
    return dtype == TB_DTYPE_F32 ? dequantize<float>(t, y, y_stride, s)
                                 : dequantize<__nv_bfloat16>(t, y, y_stride, s);
}

extern "C" int tb_b200_residual_rms_norm_mx(int dtype, const void* x, const void* residual,
                                            const void* weight, void* h_out, const TbB200Mx* y,
                                            float eps, void* stream) {
    const int rc = mx::check(y, true);
    if (rc != TB_OK) return rc;
    if (!is_float(dtype)) return TB_ERR_UNSUPPORTED_DTYPE;
    if (y->rows == 0) return TB_OK;
    if (!x) return TB_ERR_INVALID_ARG;
    cudaStream_t s = tbh::stream_of(stream);
    return dtype == TB_DTYPE_F32 ? norm<float>(x, residual, weight, h_out, y, eps, s)
                                 : norm<__nv_bfloat16>(x, residual, weight, h_out, y, eps, s);
}

extern "C" int tb_b200_swiglu_mx(int dtype, const void* gate, int64_t gate_stride, const void* up,
                                 int64_t up_stride, const TbB200Mx* out, void* stream) {
    const int rc = mx::check(out, true);
    if (rc != TB_OK) return rc;
    if (!is_float(dtype)) return TB_ERR_UNSUPPORTED_DTYPE;
    if (!strided(out->rows, out->cols, gate_stride) || !strided(out->rows, out->cols, up_stride))
        return TB_ERR_INVALID_SHAPE;
    if (out->rows == 0) return TB_OK;
    if (!gate || !up) return TB_ERR_INVALID_ARG;
    cudaStream_t s = tbh::stream_of(stream);
    return dtype == TB_DTYPE_F32
               ? swiglu<float>(gate, gate_stride, up, up_stride, out, s)
               : swiglu<__nv_bfloat16>(gate, gate_stride, up, up_stride, out, s);
}
