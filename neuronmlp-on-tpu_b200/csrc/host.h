// What the library's host sources share: the last CUDA error, the launch count,
// the device and the tensor-map encoder (defined in svdmlp.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include "../../include/svdmlp.h"

namespace svdmlp {

int cuda_fail(cudaError_t e);  // records e, returns SVDMLP_ERR_CUDA
void count_launch();
unsigned long long wait_limit_ns();
int device_sms(int* sms);  // SMs of the current device; SVDMLP_ERR_DEVICE unless it is sm_100
int planning_sms();        // the same, 148 where no device is visible
PFN_cuTensorMapEncodeTiled_v12000 encode_fn();

}  // namespace svdmlp

#define SVD_CUDA(call)                                    \
  do {                                                    \
    cudaError_t e_ = (call);                              \
    if (e_ != cudaSuccess) return svdmlp::cuda_fail(e_);  \
  } while (0)
#define SVD_CHECK(...)              \
  do {                              \
    int s_ = (__VA_ARGS__);         \
    if (s_ != SVDMLP_OK) return s_; \
  } while (0)
