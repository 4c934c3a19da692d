// Host helpers that nvfp4_api.cu shares with the library's other translation units: the
// calling thread's error text, the tensor-map encoder and the SM count.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

namespace nvfp4 {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                 const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Records `text` for nvfp4_last_error() and returns `code`.
int host_fail(int code, const char* text) noexcept;

// The same for a CUDA error of the call `what`; clears it.
int host_fail_cuda(cudaError_t error, const char* what) noexcept;

// cuTensorMapEncodeTiled, looked up once. 0 or an error already recorded.
int host_encoder(EncodeTiled* out) noexcept;

// SMs of the current device.
int host_sm_count() noexcept;

}  // namespace nvfp4
