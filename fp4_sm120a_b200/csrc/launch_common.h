// Host-side helpers shared by the launchers: status mapping, cached device
// properties.
#pragma once

#include <atomic>
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

// Whether an output of m rows of n elements (strides lda, ldb) shares memory with
// another matrix of the same sizes without being the same one: rows would be read
// after others had been written over them.  Side by side in the same rows is no
// overlap.
inline bool partly_over(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t m,
                        int64_t n, int64_t elem) {
  if (!a || !b || m < 1 || n < 1) return false;
  if (a == b && (lda == ldb || m == 1)) return false;
  using Wide = __int128;
  const Wide a0 = (Wide)(uintptr_t)a, b0 = (Wide)(uintptr_t)b;
  const Wide a1 = a0 + ((Wide)(m - 1) * lda + n) * elem, b1 = b0 + ((Wide)(m - 1) * ldb + n) * elem;
  if (a1 <= b0 || b1 <= a0) return false;
  if (lda != ldb || (b0 - a0) % elem != 0) return true;
  // Columns of b in a's rows.
  const Wide c = (((b0 - a0) / elem) % lda + lda) % lda;
  return c < n || c + n > lda;
}

// Allows KERNEL `bytes` of dynamic shared memory, once a device (asking again
// for every launch costs about as much as the launch).
template <auto KERNEL>
int allow_smem(int bytes) {
  static std::atomic<uint64_t> done;
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return cuda_status(e);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return NVFP4_OK;
  if (cudaError_t e =
          cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes))
    return cuda_status(e);
  if (dev < 64) done.fetch_or(bit, std::memory_order_release);
  return NVFP4_OK;
}

}  // namespace nvfp4
