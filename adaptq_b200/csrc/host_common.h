// What the library's translation units share on the host side (defined in adaptq_b200.cu):
// the calling thread's error string, the launch count, the failure seam and the sign generator.
#pragma once
#include <atomic>
#include <cstdint>
#include <cuda_runtime.h>

#define AQ_HIDDEN __attribute__((visibility("hidden")))

AQ_HIDDEN void aq_set_error(const char *fmt, ...);
AQ_HIDDEN void aq_clear_error();
AQ_HIDDEN void aq_count_launch();
AQ_HIDDEN cudaError_t aq_launch_status(); // of the launch just made, or an injected failure
AQ_HIDDEN void aq_sign_words(uint64_t seed, int padded, uint32_t *words, int n_words);
// Counts a launch just made and reports its failure, if any, as the error of `fn`.
inline bool aq_launched(const char *fn) {
  aq_count_launch();
  const cudaError_t e = aq_launch_status();
  if (e == cudaSuccess) return true;
  aq_set_error("%s: CUDA error: %s", fn, cudaGetErrorString(e));
  return false;
}
// SMs of a device, asked for once (148 where the driver does not tell): what grids and workspaces are sized for.
AQ_HIDDEN inline int aq_sm_count(int device) {
  static std::atomic<int> known[64] = {};
  if (device < 0 || device >= 64) return 148;
  int n = known[device].load();
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) { cudaGetLastError(); return 148; }
    known[device].store(n);
  }
  return n;
}
