// tensor_map.h -- TMA descriptors of byte tensors.
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

}  // namespace tbh
