// kv8_mma.cuh -- 8-bit codes as operands of the f16 matrix instructions.
//
// Every code is an f16 value: int8 exactly, e4m3 exactly at 2^-8 of its value
// (its exponent and mantissa bits moved into f16's places).  Conversion never
// makes a NaN or an infinity, so what lies in unused slots, multiplied by a
// weight of zero, adds nothing.
#pragma once

#include "kv8.cuh"

namespace kv8 {

// What a format's f16 operands are short of the code's value by.
template <int FORMAT>
constexpr float kOperandUnit = FORMAT == kE4m3 ? 256.0f : 1.0f;

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}

// The bytes 0 and 2 (even), and 1 and 3 (odd), of w as two f16.
template <int FORMAT>
__device__ __forceinline__ void to_f16(uint32_t w, uint32_t& even, uint32_t& odd) {
    if constexpr (FORMAT == kInt8) {
        // 1024 + (code + 128) is f16 0x6400 | code ^ 0x80; less 1152 the code
        const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        uint32_t e = (w & 0x00ff00ffu) ^ 0x64806480u;
        uint32_t o = ((w >> 8) & 0x00ff00ffu) ^ 0x64806480u;
        const __half2 he = __hsub2(*reinterpret_cast<__half2*>(&e), bias);
        const __half2 ho = __hsub2(*reinterpret_cast<__half2*>(&o), bias);
        even = *reinterpret_cast<const uint32_t*>(&he);
        odd = *reinterpret_cast<const uint32_t*>(&ho);
    } else {
        even = ((w << 8) & 0x80008000u) | ((w << 7) & 0x3f803f80u);
        odd = (w & 0x80008000u) | ((w >> 1) & 0x3f803f80u);
    }
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

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
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

}  // namespace kv8
