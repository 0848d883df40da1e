// tensor_map.cu -- TMA descriptors.  cuTensorMapEncodeTiled is the driver's:
// it is looked up through the runtime, so the library does not link libcuda.
#include "tensor_map.h"

#include <atomic>
#include <stdio.h>

#include "tb_internal.h"

namespace {
using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                            const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                            const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                            CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
std::atomic<void*> g_encode{nullptr};
}  // namespace

namespace tbh {

int encode_tiles_u8(CUtensorMap* map, const void* base, const uint64_t dims[3],
                    const uint64_t strides[2], const uint32_t box[3], int swizzle) {
    void* fn = g_encode.load();
    if (!fn) {
        cudaDriverEntryPointQueryResult found;
        TB_CUDA_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000,
                                                     cudaEnableDefault, &found));
        if (found != cudaDriverEntryPointSuccess || !fn) {
            set_error_text("cuTensorMapEncodeTiled: not in the driver");
            return TB_ERR_DEVICE;
        }
        g_encode.store(fn);
    }
    const cuuint32_t steps[3] = {1, 1, 1};
    const CUresult rc = reinterpret_cast<Encode>(fn)(
        map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base),
        reinterpret_cast<const cuuint64_t*>(dims), reinterpret_cast<const cuuint64_t*>(strides),
        box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
        swizzle == 0 ? CU_TENSOR_MAP_SWIZZLE_NONE
                     : swizzle == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
        CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) {
        char text[96];
        snprintf(text, sizeof text, "cuTensorMapEncodeTiled: CUresult %d", (int)rc);
        set_error_text(text);
        return TB_ERR_DEVICE;
    }
    return TB_OK;
}

}  // namespace tbh
