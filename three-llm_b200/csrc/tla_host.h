// Host-side helpers shared by the C ABI's translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdio.h>
#include <stdlib.h>

#include <vector>

#include "tla_internal.h"

namespace tla {

struct DeviceGuard {
  int prev = -1;
  bool moved = false;
  explicit DeviceGuard(int dev) {
    if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
    if (prev != dev) {
      cudaSetDevice(dev);
      moved = true;
    }
  }
  ~DeviceGuard() {
    if (moved && prev >= 0) cudaSetDevice(prev);
  }
};

// The status of a runtime call. A failed call's error is taken off the runtime's
// record, where a later launch's check would find it and report it as its own.
inline int from_cuda(cudaError_t e) {
  if (e == cudaSuccess) return TLA_OK;
  cudaGetLastError();
  if (getenv("TLA_DEBUG")) fprintf(stderr, "tla: CUDA error %d: %s\n", static_cast<int>(e), cudaGetErrorString(e));
  if (e == cudaErrorMemoryAllocation) return TLA_ERR_OUT_OF_MEMORY;
  return TLA_ERR_CUDA;
}

template <typename T>
int dev_alloc(T** p, size_t count) {
  *p = nullptr;
  if (count == 0) return TLA_OK;
  return from_cuda(cudaMalloc(reinterpret_cast<void**>(p), count * sizeof(T)));
}

// Checks a configuration and fills the layer's shape, RoPE and norm fields
// (no device memory); inv_freq receives the RoPE table.
int layer_params(const tla_attn_config* cfg, tla_layer* L, std::vector<float>* inv_freq);
// Device copies of the RoPE table and the norm weights (host arrays or null).
int layer_tables(tla_layer* L, const std::vector<float>& inv_freq, const float* q_norm_weight,
                 const float* k_norm_weight);

}  // namespace tla
