// Host-side helpers shared by the launchers: status mapping, cached device
// properties.
#pragma once

#include <cstddef>
#include <cstdint>
#include <cuda_runtime.h>

#include "nvfp4_b200.h"

namespace nvfp4 {

// Records the CUDA error for nvfp4_last_cuda_error() and maps it to a status.
int cuda_status(cudaError_t e);

// SM count of the current device (cached per device).  Also rejects devices
// that are not compute capability 10.0.
int device_sm_count(int* sms);

// Read (and with clear reset) the error words of the kernels in the other
// source files, for nvfp4_device_error.  The device is already synchronized.
int gemm_device_error(uint32_t* code, int clear);
int layernorm_device_error(uint32_t* code, int clear);

}  // namespace nvfp4
