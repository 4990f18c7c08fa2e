// Reading a status word and clearing it in one step: a copy and a clear in turn would lose a bit that another stream sets in between.
#include "../../include/darask_moe_b200.h"
#include <atomic>
#include "status.cuh"

namespace dmoe {

// what a call has taken, until it is copied to the host; a word is used again after so many further calls
constexpr unsigned kTaken = 256;
static __device__ unsigned g_taken[kTaken];

__global__ void status_take_kernel(unsigned* word, unsigned* taken) {
  pdl_wait();
  *taken = atomicExch(word, 0u);
}

}  // namespace dmoe

using namespace dmoe;

extern "C" int darask_status_take(unsigned* word, unsigned* host_status, cudaStream_t st) {
  if (!word || reinterpret_cast<uintptr_t>(word) % 4 || !host_status) return cudaErrorInvalidValue;
  static unsigned* known[64] = {};
  static std::atomic<unsigned> next{0};
  unsigned* taken = nullptr;
  cudaError_t e = device_word(g_taken, known, &taken);
  if (e) return e;
  taken += next++ % kTaken;
  if ((e = launch_pdl(status_take_kernel, dim3(1), dim3(1), size_t(0), st, word, taken))) return e;
  if ((e = cudaMemcpyAsync(host_status, taken, 4, cudaMemcpyDeviceToHost, st))) return e;
  return cudaStreamSynchronize(st);
}
