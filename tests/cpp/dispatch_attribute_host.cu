// Host check (no GPU is used): how much shared memory a kernel may ask for belongs to the kernel, not to a call, and calls in several threads set it at any
// time.  So the dispatch sets the same value whatever the number of experts is.
#include <cuda_runtime.h>

#include <cstdio>
#include <map>

static std::map<const void*, int> limits;
static int failures = 0, asked = 0;
template <class Kernel> cudaError_t note_attribute(Kernel kernel, cudaFuncAttribute what, int value) {
  if (what != cudaFuncAttributeMaxDynamicSharedMemorySize) return cudaSuccess;
  ++asked;
  const auto at = limits.insert({(const void*)kernel, value}).first;
  if (at->second != value) { std::printf("a limit of %d bytes, and of %d\n", at->second, value); ++failures; }
  return cudaSuccess;
}
#define cudaFuncSetAttribute note_attribute
#include "../../thrust_b200/csrc/abi_experts.cu"

void tb200_abi::call_begins(const void*) {}

int main() {
  int devices = 0;
  if (cudaGetDeviceCount(&devices) == cudaSuccess && devices > 0) { std::printf("run without a device: the addresses below are none\n"); return 1; }
  void* const buf = reinterpret_cast<void*>(256);
  for (size_t n : {(size_t)100, (size_t)100000})
    for (size_t experts : {(size_t)1, (size_t)320, (size_t)1024, (size_t)300, (size_t)1000})
      for (size_t dim : {(size_t)64, (size_t)63}) {
        size_t bytes = (size_t)1 << 30;
        if (tb200_expert_dispatch(buf, 64, buf, TB200_I32, n, 4, experts, dim, TB200_BF16, buf, (int*)buf, (int*)buf, (int*)buf, buf, &bytes, nullptr) == 0) ++failures;      // no device
      }
  return failures || !asked ? 1 : 0;
}
