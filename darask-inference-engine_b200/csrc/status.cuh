// Status words of calls that are given none: one per device and operator.
#pragma once
#include "stream_launch.cuh"

namespace dmoe {

// Address of a __device__ word on the current device, looked up once per device.
template <typename Symbol>
inline cudaError_t device_word(const Symbol& symbol, unsigned* (&known)[64], unsigned** p) {
  const int dev = current_device_slot();
  if (dev < 0) return cudaErrorInvalidDevice;
  if (!known[dev]) {
    void* q = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&q, symbol);
    if (e != cudaSuccess) return e;
    known[dev] = static_cast<unsigned*>(q);
  }
  *p = known[dev];
  return cudaSuccess;
}

}  // namespace dmoe
