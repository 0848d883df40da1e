// mx.cuh -- what the kernels of the microscaled formats share: the checked view of
// such a tensor, where its scales lie, and 32 elements to a scale and codes.
//
// A block is 32 neighbouring elements of a row.  Its scale is the least power of two
// 2^e >= 2^-127 with max|x| <= MAX 2^e (MAX 448 for e4m3, 6 for e2m1), held as the byte
// e + 127; codes are x / 2^e rounded to nearest, ties to even.  Dividing by a power of two
// is exact, so codes and scales depend on nothing but this definition.  A block with a NaN
// or an infinity has the scale 0xff, which is NaN.
#pragma once

#include <cuda_fp8.h>
#include <stdint.h>

#include "tb_device.cuh"
#include "tb_internal.h"

namespace mx {

constexpr int kE4m3 = TB_B200_MX_E4M3, kE2m1 = TB_B200_MX_E2M1;
constexpr int kTile = 128;        // columns are filled up to a multiple, rows of scales too
constexpr int kTileBytes = 512;   // scales of 128 rows and 4 blocks
constexpr uint8_t kNan = 0xff;

// A tensor as the kernels see it: rows of `pitch` bytes, `tiles` of 128 columns.
struct View {
    uint8_t* codes;
    uint8_t* scales;
    int64_t rows, pitch;
    int cols, tiles;
};

// Where the scales of row r and the four blocks of tile t lie.
__host__ __device__ __forceinline__ int64_t scales_at(int64_t r, int t, int tiles) {
    return ((r >> 7) * tiles + t) * kTileBytes + (r & 31) * 16 + (r >> 5 & 3) * 4;
}

inline int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }
inline int64_t pitch_of(int format, int64_t cols) {
    return tiles_of(cols) * kTile / (format == kE2m1 ? 2 : 1);
}

// TB_OK or the error to return.  Columns stay below 2^24 and rows below 2^31 - 128, so that
// a row's offsets and a tile's rows fit an int.
inline int check(const TbB200Mx* t, bool pointers) {
    if (!t) return TB_ERR_INVALID_ARG;
    if (t->format != kE4m3 && t->format != kE2m1) return TB_ERR_UNSUPPORTED_DTYPE;
    if (t->rows < 0 || t->rows > INT32_MAX - kTile || t->cols < 1 || t->cols > 1 << 24)
        return TB_ERR_INVALID_SHAPE;
    if (pointers && t->rows) {
        if (!t->codes || !t->scales) return TB_ERR_INVALID_ARG;
        // the product's copies: rows of 4-bit codes start on 32 bytes, scales on 16
        if ((uintptr_t)t->codes % 32 || (uintptr_t)t->scales % 16) return TB_ERR_INVALID_ARG;
    }
    return TB_OK;
}

inline View view(const TbB200Mx* t) {
    return {static_cast<uint8_t*>(t->codes), t->scales, t->rows, pitch_of(t->format, t->cols),
            (int)t->cols, (int)tiles_of(t->cols)};
}

// ------------------------------------------------------------------ codes
// The scale byte of a block whose largest magnitude has the bits `top` (f32's, without the
// sign): 448 is 1.75 * 2^8 and 6 is 1.5 * 2^2, so e is top's exponent less 8 or 2, and one
// more where its mantissa is above that.
template <int FORMAT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) {
    constexpr uint32_t kMost = FORMAT == kE4m3 ? 0x600000u : 0x400000u;
    constexpr int kDown = FORMAT == kE4m3 ? 8 : 2;
    const int e = (int)(top >> 23) - kDown + ((top & 0x7fffffu) > kMost);
    return top >= 0x7f800000u ? kNan : (uint32_t)max(e, 0);
}
// What elements are multiplied with to become codes: 2^-e; NaN for a block that is NaN.
__device__ __forceinline__ float inverse_of(uint32_t byte) {
    return byte == kNan ? __uint_as_float(0x7fffffffu) : __uint_as_float((254u - byte) << 23);
}
// A scale's value.
__device__ __forceinline__ float value_of(uint32_t byte) {
    return byte == 0    ? __uint_as_float(1u << 22)  // 2^-127
           : byte == kNan ? __uint_as_float(0x7fffffffu)
                          : __uint_as_float(byte << 23);
}

// Four scaled elements as e4m3 codes, eight as e2m1 codes, the first in the low bits.
__device__ __forceinline__ uint32_t e4m3x4(const float* v) {
    uint32_t w;
    asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n"
        " cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n mov.b32 %0, {l, h};\n}"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
    return w;
}
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
    uint32_t w;
    asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
        " cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}

// Four elements as e2m1 codes.
__device__ __forceinline__ uint16_t e2m1x4(const float* v) {
    uint16_t w;
    asm("{\n .reg .b8 a, b;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n mov.b16 %0, {a, b};\n}"
        : "=h"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]));
    return w;
}

// E neighbouring elements of a row, E = 4, 8 or 16, to codes and scales: the 32 / E lanes of a
// block and the 128 / E lanes of a tile are neighbours in a warp.  Chunk c of row r; every
// lane of the warp calls it, `live` or not.
template <int FORMAT, int E>
__device__ __forceinline__ void store_block(const View& out, int64_t r, int c, bool live,
                                            float (&v)[E]) {
    constexpr int kBlock = 32 / E, kLanes = 128 / E;
    float most = 0.0f;  // a NaN stays one, and its bits are the largest
#pragma unroll
    for (int i = 0; i < E; i += 2)
        asm("max.NaN.f32 %0, %1, %2, %3;"
            : "=f"(most)
            : "f"(most), "f"(fabsf(v[i])), "f"(fabsf(v[i + 1])));
    uint32_t top = __float_as_uint(most);
#pragma unroll
    for (int o = 1; o < kBlock; o <<= 1) top = max(top, __shfl_xor_sync(tbk::kFull, top, o));
    const uint32_t byte = scale_byte<FORMAT>(top);
    const int lane = threadIdx.x & 31;
    uint32_t four = byte << 8 * (lane / kBlock % 4);
#pragma unroll
    for (int o = kBlock; o < kLanes; o <<= 1) four |= __shfl_xor_sync(tbk::kFull, four, o);
    if (!live) return;
    const float by = inverse_of(byte);
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] *= by;
    uint8_t* to = out.codes + r * out.pitch + (int64_t)c * (FORMAT == kE4m3 ? E : E / 2);
    if constexpr (FORMAT == kE4m3 && E == 16)
        *reinterpret_cast<uint4*>(to) =
            make_uint4(e4m3x4(v), e4m3x4(v + 4), e4m3x4(v + 8), e4m3x4(v + 12));
    else if constexpr (FORMAT == kE4m3 && E == 8)
        *reinterpret_cast<uint2*>(to) = make_uint2(e4m3x4(v), e4m3x4(v + 4));
    else if constexpr (FORMAT == kE4m3)
        *reinterpret_cast<uint32_t*>(to) = e4m3x4(v);
    else if constexpr (E == 16)
        *reinterpret_cast<uint2*>(to) = make_uint2(e2m1x8(v), e2m1x8(v + 8));
    else if constexpr (E == 8)
        *reinterpret_cast<uint32_t*>(to) = e2m1x8(v);
    else
        *reinterpret_cast<uint16_t*>(to) = e2m1x4(v);
    if (lane % kLanes == 0)
        *reinterpret_cast<uint32_t*>(out.scales + scales_at(r, c / kLanes, out.tiles)) = four;
}

}  // namespace mx
