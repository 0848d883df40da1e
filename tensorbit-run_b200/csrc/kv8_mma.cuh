// kv8_mma.cuh -- 8-bit codes as operands of the f16 matrix instructions.
//
// Every code is an f16 value exactly, subnormal e4m3 codes among them.
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

// Which elements of a word of four the two registers of word() hold.
template <int FORMAT>
__device__ constexpr int word_element(int reg, int i) {
    return FORMAT == kInt8 ? reg + 2 * i : 2 * reg + i;
}
template <int FORMAT>
__device__ __forceinline__ void word(uint32_t w, uint32_t& r0, uint32_t& r1) {
    if constexpr (FORMAT == kInt8) {
        r0 = int8_pair(w);
        r1 = int8_pair(w >> 8);
    } else {
        r0 = e4m3_pair(w, false);
        r1 = e4m3_pair(w, true);
    }
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
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

// 16 consecutive elements as f32, the first `n` of them (a multiple of 16: all or none).
template <typename T>
__device__ __forceinline__ void load16(const T* p, bool live, bool vec, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = 0.0f;
    if (!live) return;
    if (vec) {
        constexpr int V = tbk::Elt<T>::kVec;
#pragma unroll
        for (int i = 0; i < 16; i += V) {
            float x[V];
            tbk::load_vec<T, V>(p + i, x);
#pragma unroll
            for (int e = 0; e < V; ++e) v[i + e] = x[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = tbk::Elt<T>::load(p + i);
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
// 128, with the swizzle of that width; past head_dim zeros are loaded).
inline int tile_map(CUtensorMap* map, const TbB200Kv8* c, const void* codes, int width, int keys) {
    const uint64_t dims[3] = {(uint64_t)c->head_dim, (uint64_t)c->page,
                              (uint64_t)(c->n_pages > 0 ? c->n_pages : 1) * c->n_kv_heads};
    const uint64_t strides[2] = {(uint64_t)c->head_dim, (uint64_t)c->head_dim * c->page};
    const uint32_t box[3] = {(uint32_t)width, (uint32_t)keys, 1};
    return tbh::encode_tiles_u8(map, codes, dims, strides, box, width);
}

}  // namespace kv8
