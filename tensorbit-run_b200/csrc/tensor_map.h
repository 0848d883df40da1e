// tensor_map.h -- TMA descriptors of tensors of bytes and of 4-bit elements.
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace tbh {

// A 3-D tensor of bytes at `base` (dims innermost first; strides in bytes of
// the outer two dimensions) in tiles of `box`, placed in shared memory with the
// swizzle of `swizzle` (64, 128 or, for none, 0) bytes; elements out of range read as zero.
// TB_OK, or TB_ERR_DEVICE with the reason recorded.
int encode_tiles_u8(CUtensorMap* map, const void* base, const uint64_t dims[3],
                    const uint64_t strides[2], const uint32_t box[3], int swizzle);
// The same of 4-bit elements, two to a byte: 16 of them become 8 bytes and 8 bytes of fill
// in shared memory, as the matrix instructions take them beside 8-bit ones.  dims[0] and the
// innermost coordinate of a copy are multiples of 128, box[0] is 128, base and strides are
// multiples of 32 bytes, and the swizzle is 128 or 0.
int encode_tiles_u4(CUtensorMap* map, const void* base, const uint64_t dims[3],
                    const uint64_t strides[2], const uint32_t box[3], int swizzle);

}  // namespace tbh
