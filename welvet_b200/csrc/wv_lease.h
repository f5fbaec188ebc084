// Device scratch of a call (wv_gemm_tcgen05.cu): a buffer of the stream's own, or of the graph's in a capture, valid until later
// work on that stream takes it again. The lease is kept while the call enqueues the kernels that use it.
#pragma once
#include <cuda_runtime.h>
#include <mutex>

struct WvLease {
  float* p = nullptr;
  bool free_after = false;
  cudaStream_t free_on = nullptr;
  std::unique_lock<std::mutex> lock;
  ~WvLease() { if (free_after) cudaFreeAsync(p, free_on); }
};
int wv_lease(WvLease& out, size_t floats, cudaStream_t st, const char* what);     // WV_OK, or WV_ENOMEM with `what` in the message
