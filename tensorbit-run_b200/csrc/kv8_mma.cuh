// kv8_mma.cuh -- 8-bit codes as operands of the matrix instructions: as they
// are (int8 x int8), or as f16, which holds every code exactly, subnormal e4m3
// codes among them.
#pragma once

#include <atomic>

#include "kv8.cuh"
#include "tma.cuh"
#include "tensor_map.h"

namespace kv8 {

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}

// Two codes (the low or high half of w) as two f16.
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w, bool high) {
    uint32_t r;
    const uint16_t h = (uint16_t)(high ? w >> 16 : w);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(h));
    return r;
}
// Bytes 0 and 2 of w (1 and 3: of w >> 8): 1024 + (code + 128) is the f16
// 0x6400 | (code ^ 0x80); less 1152 it is the code.
__device__ __forceinline__ uint32_t int8_pair(uint32_t w) {
    uint32_t e = (w & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&e), bias);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Elements 0 .. 3 of two words, each with its partner of the other word.
template <int FORMAT>
__device__ __forceinline__ void words(uint32_t a, uint32_t b, uint32_t (&r)[4]) {
    if constexpr (FORMAT == kInt8) {
        const uint32_t x = prmt(a, b, 0x5410), y = prmt(a, b, 0x7632);
        r[0] = int8_pair(x);
        r[1] = int8_pair(x >> 8);
        r[2] = int8_pair(y);
        r[3] = int8_pair(y >> 8);
    } else {
        const uint32_t x = prmt(a, b, 0x5140), y = prmt(a, b, 0x7362);
        r[0] = e4m3_pair(x, false);
        r[1] = e4m3_pair(x, true);
        r[2] = e4m3_pair(y, false);
        r[3] = e4m3_pair(y, true);
    }
}

// The left operand of mma_codes from shared memory: lane i gives the address of
// the 16 bytes of row i % 16 and half i / 16 of 32.
__device__ __forceinline__ void load_operand(uint32_t addr, uint32_t (&w)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "r"(addr)
                 : "memory");
}

// The transpose of an 8 x 8 tile of f16, two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// d += a b: a 16 x 16 row-major, b 16 x 8 column-major, f32 sums.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a b + c of int8 codes, 32 elements deep, exact.
__device__ __forceinline__ void mma_codes(int (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                          uint32_t b1, const int (&c)[4]) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%11,%12,%13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]),
          "r"(c[3]));
}

// A row of q as operands against the codes, kRegs registers for four elements:
//   int8: the nearest whole number to q * 127 * 2^14 / top as three digits of
//     radix 128 (2^-22 of top, the row's largest);
//   e4m3: q * 2^k (top in [2^14, 2^15)) as f16, an f32 row as two (hi + lo): a
//     bf16 element exactly, an f32 one to 2^-22 of itself, or either to 2^-39 of
//     top where that is larger.  An e4m3 product of mma.sync costs its operands'
//     conversions to f16 for each 8 rows and each part of q, and a sum of its
//     own; f16 products need a key's codes converted once (a step of 32 keys, 16
//     rows and 64 elements took 644 warp instructions with two e4m3 parts).
template <typename T, int FORMAT>
struct QParts {
    static constexpr int kParts = FORMAT == kInt8 ? 3 : sizeof(T) == 4 ? 2 : 1;
    static constexpr int kRegs = FORMAT == kInt8 ? 3 : 2 * kParts;
    float lift, unit;  // q's factor; what a sum of products is to be multiplied with

    __device__ explicit QParts(float top) {
        if constexpr (FORMAT == kInt8) {
            lift = 2080768.0f / fmaxf(top, 7.8886090522101181e-31f);
            unit = fmaxf(top, 7.8886090522101181e-31f) * (1.0f / 2080768.0f);
        } else {
            const int e = min(max((int)(__float_as_uint(top) >> 23), 20), 254);
            lift = __uint_as_float((uint32_t)(127 + 14 - e + 127) << 23);
            unit = __uint_as_float((uint32_t)(e - 14) << 23);
        }
    }
    // Four elements: int8 a word of each digit, e4m3 two pairs of each part.
    __device__ void split(const float* x, uint32_t (&w)[kRegs]) const {
        if constexpr (FORMAT == kInt8) {
#pragma unroll
            for (int p = 0; p < 3; ++p) w[p] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = __float2int_rn(x[i] * lift);
                const int a = (v + 8192) >> 14, r = v - (a << 14), b = (r + 64) >> 7;
                w[0] |= (uint32_t)(a & 0xff) << 8 * i;
                w[1] |= (uint32_t)(b & 0xff) << 8 * i;
                w[2] |= (uint32_t)((r - (b << 7)) & 0xff) << 8 * i;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float a = x[2 * i] * lift, b = x[2 * i + 1] * lift;
                w[i] = pack_f16x2(a, b);
                if constexpr (kParts == 2) {
                    const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    w[2 + i] = pack_f16x2(a - u.x, b - u.y);
                }
            }
        }
    }
};

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// One tile of a 3-D tensor map into shared memory, its bytes counted on bar.
__device__ __forceinline__ void tma_load3(void* dst, const CUtensorMap* map, int x, int y, int z,
                                          uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(tbk::smem_addr(dst)),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(tbk::smem_addr(bar))
        : "memory");
}

// Four consecutive elements as f32, zeros if not live; vec: aligned to all four.
template <typename T>
__device__ __forceinline__ void load4(const T* p, bool live, bool vec, float (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0.0f;
    if (!live) return;
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = tbk::Elt<T>::load(p + i);
    } else if constexpr (sizeof(T) == 4) {
        tbk::load_vec<T, 4>(p, v);
    } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(w.x << 16);
        v[1] = __uint_as_float(w.x & 0xffff0000u);
        v[2] = __uint_as_float(w.y << 16);
        v[3] = __uint_as_float(w.y & 0xffff0000u);
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, const float (&v)[4]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 4; ++i) tbk::Elt<T>::store(p + i, v[i]);
    } else if constexpr (sizeof(T) == 4) {
        tbk::store_vec<T, 4>(p, v);
    } else {
        *reinterpret_cast<uint2*>(p) =
            make_uint2(tbk::pack_bf16x2(v[0], v[1]), tbk::pack_bf16x2(v[2], v[3]));
    }
}

// Run `set` (a CUDA call for the current device) unless it has been: `done` has
// a bit per device.
template <typename F>
int once_per_device(std::atomic<uint64_t>& done, F set) {
    const tbh::DeviceState* ds = tbh::current_device_state();
    if (!ds) return TB_ERR_DEVICE;
    const uint64_t bit = 1ull << ds->device;
    if (done.load() & bit) return TB_OK;
    TB_CUDA_TRY(set());
    done.fetch_or(bit);
    return TB_OK;
}

// The cache's codes as tiles of `keys` keys of one page by `width` bytes (64 or
// 128, with the swizzle of that width or none; past head_dim zeros are loaded).
inline int tile_map(CUtensorMap* map, const TbB200Kv8* c, const void* codes, int width, int keys,
                    bool swizzled = true) {
    const uint64_t dims[3] = {(uint64_t)c->head_dim, (uint64_t)c->page,
                              (uint64_t)c->n_pages * c->n_kv_heads};
    const uint64_t strides[2] = {(uint64_t)c->head_dim, (uint64_t)c->head_dim * c->page};
    const uint32_t box[3] = {(uint32_t)width, (uint32_t)keys, 1};
    return tbh::encode_tiles_u8(map, codes, dims, strides, box, swizzled ? width : 0);
}

}  // namespace kv8
