// matrix_host.h -- what the block-scaled matrices (fp8.cu, fp4.cu) share on the
// host: sources on other devices, tensor maps of bytes.
#pragma once
#include "host_util.h"
#include "umma_host.h"

namespace qrm {
namespace {

// waits for what any stream still writes at p, when that is on another device
cudaError_t await_source(const void* p, int device) {
    cudaPointerAttributes at{};
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();   // the copy will say what is wrong with it
        return cudaSuccess;
    }
    if (at.type != cudaMemoryTypeDevice || at.device == device) return cudaSuccess;
    DeviceGuard there;
    const cudaError_t e = there.enter(at.device);
    return e == cudaSuccess ? cudaDeviceSynchronize() : e;
}

// 8-bit tensor of up to five dimensions, innermost first, as a TMA map; what
// lies outside reads as zero
bool encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
    auto fn = tensor_map_encoder();
    if (!fn) return false;
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kSmemMost = 227 * 1024;

}  // namespace
}  // namespace qrm
