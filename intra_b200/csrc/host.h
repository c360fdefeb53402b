// Host helpers shared by the translation units behind the C ABI: error reporting, the current device, argument checks.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/intra_b200.h"

namespace intra {

extern thread_local int g_last_cuda_error;      // capi.cu

// The current device's status word of the kernels of serving.cu.
cudaError_t serving_status_word(int** word);

constexpr int MAX_DEVICES = 64;

// Every failure is reported once: the runtime's own record of it is cleared, or the check after the next launch
// would report it again.
inline int cuda_fail(cudaError_t e) {
  g_last_cuda_error = static_cast<int>(e);
  cudaGetLastError();
  return INTRA_ERR_CUDA;
}

struct DeviceGuard {
  int prev = -1;
  bool ok = true;
  explicit DeviceGuard(int device) {
    if (cudaGetDevice(&prev) != cudaSuccess) { ok = false; return; }
    if (prev != device && cudaSetDevice(device) != cudaSuccess) ok = false;
  }
  ~DeviceGuard() {
    int cur = -1;
    if (prev >= 0 && cudaGetDevice(&cur) == cudaSuccess && cur != prev) cudaSetDevice(prev);
  }
};

// Shared-memory opt-in of a kernel, on the current device. Allocates nothing.
template <typename K>
cudaError_t opt_in_smem(K kernel, int bytes) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace intra
