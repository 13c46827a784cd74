// Stream-ordered scratch buffer: taken from the device's memory pool on the
// launching stream and returned to it (also stream-ordered) when the object
// goes out of scope, so kernels already queued on the stream keep a valid
// buffer and other streams never see it.
#pragma once
#include "common.cuh"

namespace mt {
int scratch_pool(cudaMemPool_t* pool);   // the library's own on the current device, which keeps what is freed
enum class Scratch { kDevicePool, kOwnPool };

struct TempBuf {
  void* ptr = nullptr;
  cudaStream_t st;
  bool ok_ = true;
  TempBuf(size_t bytes, cudaStream_t s, Scratch from = Scratch::kDevicePool) : st(s) {
    if (bytes == 0) return;
    cudaMemPool_t pool;
    if (from == Scratch::kOwnPool && scratch_pool(&pool) != MT_OK) { ok_ = false; return; }
    cudaError_t e = from == Scratch::kOwnPool ? cudaMallocFromPoolAsync(&ptr, bytes, pool, s) : cudaMallocAsync(&ptr, bytes, s);
    if (e != cudaSuccess) {
      set_error("scratch allocation of %zu bytes failed: %s", bytes, cudaGetErrorString(e));
      ok_ = false;
      ptr = nullptr;
    }
  }
  ~TempBuf() { if (ptr) cudaFreeAsync(ptr, st); }
  bool ok() const { return ok_; }
  TempBuf(const TempBuf&) = delete;
  TempBuf& operator=(const TempBuf&) = delete;
};
}  // namespace mt
