// Host helpers of the C entry points shared between translation units (capi.cu holds
// them): the error message of the calling thread, the tensor-map encoder, SM counts.
#pragma once
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include "../../include/tttj_b200.h"

namespace tttj {

int capi_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int capi_cuda_fail(cudaError_t e, const char* what);
PFN_cuTensorMapEncodeTiled_v12000 capi_encode_fn();
int capi_sm_count(int device);

}  // namespace tttj

#define CAPI_CUDA(call)                                        \
  do {                                                         \
    cudaError_t e_ = (call);                                   \
    if (e_ != cudaSuccess) return tttj::capi_cuda_fail(e_, #call); \
  } while (0)
