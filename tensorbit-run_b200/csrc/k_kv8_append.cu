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
// HBM bound: the rows read once, one byte an element written.  A unit is (page
// that gets rows, head), its K and V; which pages those are is on the device, so the
// grid has a slot for each page that could: a sequence's rows from s to e touch at
// most e / page - s / page + 2 pages, so sequence i's slots start at row_start[i] /
// page + 2 i, which a warp finds its sequence by.
//
// A unit has the warps, up to a CTA's 8, that hold its page's rows when prompts fill
// it, one warp (and a CTA 8 heads) when a call brings few rows a sequence: then the
// time is the chain of loads that leads to the rows, and a token's 16 vectors of a
// head need no more lanes.  The rows stay in registers between amax and the codes, up
// to kHold vectors a thread (a page of 64 rows of 128 in bf16); what is past that is
// read again, a vector at a time: such prompts in pages of 128 take 30 us and in f32,
// pages of 64, 37 (their bytes: 17 and 23).  The rule goes by the call's mean rows a
// sequence: 1500 rows beside 255 single tokens, all in one warp a unit, take 21 us, and
// 4.1 and 4.3 as two calls.
//
// Measured, 8 heads of 128, bf16: 14476 tokens of five prompts, e4m3, 17.1 us,
// 5.2 TB/s (18.3 with three CTAs an SM); 256 sequences' token, int8, 4.2 us, a launch
// and the chain row_start -> page and rows -> scale and code.  At four CTAs an SM (64
// registers) the forms of two and four warps a unit, for small pages, spill some 45
// bytes a thread, with which their times below were measured.
#include "kv8.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kHold = 4;
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

// V elements of a row: their largest magnitude (as bits, which order like the
// values; NaN and infinity are kInf or above) and their codes.
template <typename T, int V>
struct Piece {
    T e[V];
    static __device__ Piece load(const T* p) {
        Piece x;
#pragma unroll
        for (int i = 0; i < V; ++i) x.e[i] = p[i];
        return x;
    }
    __device__ float at(int i) const { return tbk::Elt<T>::load(&e[i]); }
};
template <>
struct Piece<float, 4> {
    uint4 w;
    static __device__ Piece load(const float* p) {
        return {__ldcs(reinterpret_cast<const uint4*>(p))};
    }
    __device__ float at(int i) const { return __uint_as_float((&w.x)[i]); }
};
template <>
struct Piece<__nv_bfloat16, 8> {
    uint4 w;
    static __device__ Piece load(const __nv_bfloat16* p) {
        return {__ldcs(reinterpret_cast<const uint4*>(p))};
    }
    __device__ float at(int i) const {
        const uint32_t x = (&w.x)[i / 2];
        return __uint_as_float(i % 2 ? x & 0xffff0000u : x << 16);
    }
};

constexpr uint32_t kInf = 0x7f800000u;

template <typename T, int V>
__device__ __forceinline__ uint32_t top_of(const Piece<T, V>& x) {
    uint32_t top = 0;
    if constexpr (sizeof(T) == 2 && V == 8) {  // two magnitudes a word
        const uint32_t m = 0x7fff7fffu;
        top = __vmaxu2(__vmaxu2(x.w.x & m, x.w.y & m), __vmaxu2(x.w.z & m, x.w.w & m));
        return max(top & 0xffff0000u, top << 16);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, __float_as_uint(x.at(i)) & 0x7fffffffu);
        return top;
    }
}

// The codes of x * per; FINITE: of finite values, whose products are within the
// format's range.
template <int FORMAT, bool FINITE, typename T, int V>
__device__ __forceinline__ void store_codes(uint8_t* p, const Piece<T, V>& x, float per) {
    constexpr float most = FORMAT == kv8::kInt8 ? 127.0f : 448.0f;
    float v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        v[i] = x.at(i);
        if (!FINITE) {
            v[i] *= per;
            v[i] = v[i] != v[i] ? 0.0f : fminf(fmaxf(v[i], -most), most);
        }
    }
    const float f = FINITE ? per : 1.0f;
    uint32_t w[(V + 3) / 4] = {};
    if constexpr (FORMAT == kv8::kInt8) {
        // the sum with 1.5 * 2^23 rounds to a whole number, its low byte the code
        uint32_t u[V];
#pragma unroll
        for (int i = 0; i < V; ++i) u[i] = __float_as_uint(fmaf(v[i], f, 12582912.0f));
        if constexpr (V >= 4) {
#pragma unroll
            for (int i = 0; i < V; i += 4)
                w[i / 4] = __byte_perm(__byte_perm(u[i], u[i + 1], 0x0040),
                                       __byte_perm(u[i + 2], u[i + 3], 0x0040), 0x5410);
        } else {
            w[0] = u[0] & 0xff;
        }
    } else if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 2)
            w[i / 4] |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[i] * f, v[i + 1] * f),
                                                           __NV_SATFINITE, __NV_E4M3)
                        << 8 * (i % 4);
    } else {
        w[0] = kv8::encode<FORMAT>(v[0] * f);
    }
    if constexpr (V == 8)
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else if constexpr (V == 4)
        *reinterpret_cast<uint32_t*>(p) = w[0];
    else
        *p = (uint8_t)w[0];
}

template <typename T, int FORMAT, int V, int WARPS>  // WARPS of a unit
__global__ void __launch_bounds__(kThreads, WARPS == 1 ? 3 : 4) k_append(const __grid_constant__ Args a) {
    __shared__ uint2 red[kThreads / 32];
    constexpr int kUnit = 32 * WARPS;  // threads
    const kv8::Batch& b = a.b;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x % kUnit;
    const int slot = blockIdx.x, page = 1 << b.page_shift;
    const int head = blockIdx.y * (kThreads / kUnit) + threadIdx.x / kUnit;
    if (head >= a.hkv) return;  // whole warps of units of one warp
    kv8::Seq s;
    const int seq = kv8::find_sequence(
        b, slot, [&](int lo, int i) { return (lo >> b.page_shift) + 2 * i; }, s);
    const int first = max(s.first, 0);  // rows before position 0 are padding
    const int logical = (first >> b.page_shift) + slot - ((s.lo >> b.page_shift) + 2 * seq);
    const int64_t begin = (int64_t)logical << b.page_shift;
    // (a slot before the first sequence's, where row_start[0] > 0, has no page)
    if (s.n == 0 || logical < first >> b.page_shift || begin >= s.len) return;
    if (logical >= b.width) {
        if (tid == 0) atomicOr(a.status, TB_B200_FLAG_POSITION_RANGE);
        return;
    }
    const int id = b.table[seq * b.table_stride + logical];
    // slots [from, to) of the page are new; slot from is row `row`
    const int from = max(first - (int)begin, 0);
    const int to = (int)min((int64_t)page, s.len - begin);
    const int row = s.lo + (int)(begin + from - s.first);
    const int64_t strides[2] = {a.k_stride, a.v_stride};
    const T* x[2] = {static_cast<const T*>(a.k) + row * a.k_stride + (int64_t)head * a.d,
                     static_cast<const T*>(a.v) + row * a.v_stride + (int64_t)head * a.d};

    // pieces tid, tid + kUnit, .. of the new rows, `per_row` of them a row
    const int per_row = a.d / V, n = (to - from) * per_row;
    const int down = kUnit / per_row, right = kUnit - down * per_row;
    const int r0 = tid / per_row, c0 = tid - r0 * per_row;
    int r = r0, c = c0;
    auto next = [&] {
        r += down;
        c += right;
        if (c >= per_row) {
            c -= per_row;
            ++r;
        }
    };
    auto piece = [&](int kv) { return Piece<T, V>::load(x[kv] + r * strides[kv] + c * V); };
    Piece<T, V> hold[2][kHold];
#pragma unroll
    for (int u = 0; u < kHold; ++u) {
        if (tid + u * kUnit < n) {
            hold[0][u] = piece(0);
            hold[1][u] = piece(1);
        }
        next();
    }
    const int r_rest = r, c_rest = c;
    if (id < 0 || id >= b.n_pages) {
        if (tid == 0) atomicOr(a.status, TB_B200_FLAG_PAGE_RANGE);
        return;
    }
    const int64_t unit = (int64_t)id * a.hkv + head;
    uint8_t* codes[2] = {a.k_codes + (unit << b.page_shift) * a.d,
                         a.v_codes + (unit << b.page_shift) * a.d};
    const float old[2] = {from > 0 ? a.k_scale[unit] : 0.0f, from > 0 ? a.v_scale[unit] : 0.0f};
    uint32_t top[2] = {0, 0};
#pragma unroll
    for (int u = 0; u < kHold; ++u)
        if (tid + u * kUnit < n) {
            top[0] = max(top[0], top_of(hold[0][u]));
            top[1] = max(top[1], top_of(hold[1][u]));
        }
    for (int i = tid + kHold * kUnit; i < n; i += kUnit) {
        top[0] = max(top[0], top_of(piece(0)));
        top[1] = max(top[1], top_of(piece(1)));
        next();
    }
    auto over_unit = [&] {
        top[0] = __reduce_max_sync(tbk::kFull, top[0]);
        top[1] = __reduce_max_sync(tbk::kFull, top[1]);
        if (WARPS == 1) return;
        const int in_cta = warp / WARPS;  // the unit's place in the CTA
        auto meet = [&] {
            asm volatile("bar.sync %0, %1;" ::"r"(in_cta + 1), "n"(kUnit) : "memory");
        };
        meet();
        if (lane == 0) red[warp] = make_uint2(top[0], top[1]);
        meet();
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
            top[0] = max(top[0], red[in_cta * WARPS + i].x);
            top[1] = max(top[1], red[in_cta * WARPS + i].y);
        }
    };
    over_unit();
    const bool finite = max(top[0], top[1]) < kInf;
    if (!finite) {  // the largest of the finite ones
        if (tid == 0) atomicOr(a.status, TB_B200_FLAG_NONFINITE);
        top[0] = top[1] = 0;
        r = r0;
        c = c0;
        for (int i = tid; i < n; i += kUnit) {
            for (int kv = 0; kv < 2; ++kv) {
                const Piece<T, V> y = piece(kv);
                for (int e = 0; e < V; ++e) {
                    const uint32_t bits = __float_as_uint(y.at(e)) & 0x7fffffffu;
                    if (bits < kInf) top[kv] = max(top[kv], bits);
                }
            }
            next();
        }
        over_unit();
    }
    float now[2], per[2];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        now[kv] = fmaxf(scale_for<FORMAT>(__uint_as_float(top[kv])), old[kv]);
        per[kv] = 1.0f / now[kv];  // both powers of two: exact
        if (!(now[kv] > old[kv] && from > 0)) continue;
        const float ratio = old[kv] * per[kv];
        uint4* held = reinterpret_cast<uint4*>(codes[kv]);
        for (int i = tid; i < from * a.d / 16; i += kUnit) {  // d is a multiple of 16
            uint4 w = held[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t y = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y |= (uint32_t)kv8::encode<FORMAT>(
                             kv8::decode<FORMAT>((uint8_t)((&w.x)[j] >> 8 * e)) * ratio)
                         << 8 * e;
                (&w.x)[j] = y;
            }
            held[i] = w;
        }
    }
    auto store = [&](auto finite) {
        auto put = [&](int kv, const Piece<T, V>& y) {
            store_codes<FORMAT, finite.value>(codes[kv] + (from + r) * a.d + c * V, y, per[kv]);
        };
        r = r0;
        c = c0;
#pragma unroll
        for (int u = 0; u < kHold; ++u) {
            if (tid + u * kUnit < n) {
                put(0, hold[0][u]);
                put(1, hold[1][u]);
            }
            next();
        }
        r = r_rest;
        c = c_rest;
        for (int i = tid + kHold * kUnit; i < n; i += kUnit) {
            put(0, piece(0));
            put(1, piece(1));
            next();
        }
    };
    if (finite)
        store(std::true_type{});
    else
        store(std::false_type{});
    if (WARPS == 1) __syncwarp();  // every thread has read the scales (else: over_unit's barriers)
    if (tid == 0) {
        a.k_scale[unit] = now[0];
        a.v_scale[unit] = now[1];
    }
}

template <typename T, int FORMAT, int V, int WARPS>
void launch_units(const Args& a, unsigned slots, cudaStream_t s) {
    constexpr int kUnits = kThreads / 32 / WARPS;  // of a CTA
    const unsigned heads = (unsigned)(a.hkv + kUnits - 1) / kUnits;
    k_append<T, FORMAT, V, WARPS><<<dim3(slots, heads), kThreads, 0, s>>>(a);
}

template <typename T, int FORMAT, int V>
void launch(const Args& a, int warps, unsigned slots, cudaStream_t s) {
    if (warps == 1)
        launch_units<T, FORMAT, V, 1>(a, slots, s);
    else if (warps == 2)
        launch_units<T, FORMAT, V, 2>(a, slots, s);
    else if (warps == 4)
        launch_units<T, FORMAT, V, 4>(a, slots, s);
    else
        launch_units<T, FORMAT, V, 8>(a, slots, s);
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
    const unsigned slots = (unsigned)(batch->rows / cache->page + 2 * batch->n_seqs);
    // One warp a unit when a sequence brings so few rows that kHold vectors a
    // lane hold them (bf16: rows * d <= 1024 elements).  A warp and a CTA a unit, 8
    // heads of 128: 256 sequences' token 4.7 and 15.1 us, 64 of 8 tokens 4.5 and 7.3,
    // of 16 7.2 and 7.2, of 32 16.7 and 8.4.  Else as many as hold a page: 14500 tokens
    // in pages of 16, heads of 128, two warps 21.9 us, eight 36.5; heads of 64, one
    // 10.6, eight 32.9; pages of 32, four 21.6, eight 23.1.
    const size_t size = dtype == TB_DTYPE_F32 ? 4 : 2;
    const int64_t few = 32 * kHold * 16;  // bytes that a warp's lanes hold
    int warps = 1;
    if (batch->rows * cache->head_dim * (int64_t)size > batch->n_seqs * few)
        while (warps < 8 && cache->page * cache->head_dim * (int64_t)size > warps * few) warps *= 2;
    const bool vec = tbh::aligned16(k) && tbh::aligned16(v) && k_stride * size % 16 == 0 &&
                     v_stride * size % 16 == 0;
    cudaStream_t s = tbh::stream_of(stream);
    const bool f32 = dtype == TB_DTYPE_F32, int8 = cache->format == kv8::kInt8;
    if (f32 && int8)
        vec ? launch<float, kv8::kInt8, 4>(a, warps, slots, s)
            : launch<float, kv8::kInt8, 1>(a, warps, slots, s);
    else if (f32)
        vec ? launch<float, kv8::kE4m3, 4>(a, warps, slots, s)
            : launch<float, kv8::kE4m3, 1>(a, warps, slots, s);
    else if (int8)
        vec ? launch<__nv_bfloat16, kv8::kInt8, 8>(a, warps, slots, s)
            : launch<__nv_bfloat16, kv8::kInt8, 1>(a, warps, slots, s);
    else
        vec ? launch<__nv_bfloat16, kv8::kE4m3, 8>(a, warps, slots, s)
            : launch<__nv_bfloat16, kv8::kE4m3, 1>(a, warps, slots, s);
    TB_LAUNCH_CHECK("8-bit cache append kernel");
    return TB_OK;
}
