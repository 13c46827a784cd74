// The paged key/value cache: what its kernels share (see mytorch_b200.h for the layout).
#pragma once
#include "common.cuh"
#include <atomic>

namespace mt {

constexpr int kPagedFlag = 3;            // device status: no page left, or a page or slot outside the pool

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, Division by Invariant Integers
// using Multiplication, 1994): m = floor(2^32 (2^s - d) / d) + 1 with 2^s >= d.
struct FastDiv {
  uint32_t d, m, s;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), s(0) {
    while (s < 32 && (1ull << s) < div) ++s;
    m = (uint32_t)((((1ull << s) - div) << 32) / div + 1);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(m, n) + n) >> s; }
};

// A kernel's limit on dynamic shared memory, raised once per device (racing first calls raise it twice, harmlessly).
struct SmemLimit {
  std::atomic<bool> done[16] = {};
  int raise(const void* kern, int bytes) {
    int dev = 0;
    MT_CHECK_CUDA(cudaGetDevice(&dev));
    if (dev >= 0 && dev < 16 && done[dev].load(std::memory_order_acquire)) return MT_OK;
    MT_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev >= 0 && dev < 16) done[dev].store(true, std::memory_order_release);
    return MT_OK;
  }
};

struct PagedAttnParams {
  const void *q, *kp, *vp;
  void* o;
  mt_strides3 sq, sc, so;                // q, o: {-, head, row}; pools: {page, head, row}
  const int32_t *tables, *starts, *kv_len;
  int requests, width, rows, heads, kv_heads, group, n_pages;
  int least_rows, most_rows;             // query rows per key/value head of the requests that a launch works on
  FastDiv page, by_group;
  float scale_log2;
  int q_pairs, o_quads;                  // rows of q on 4-byte, rows of o on 8-byte (16-byte in fp32) boundaries
  int* flag;
};

// One request as the attention kernels see it. `past` may be negative (fewer keys than new rows: the
// first rows see nothing).
struct PagedRequest {
  int q0, n_new, past, keys;
};

__device__ __forceinline__ PagedRequest paged_request(const PagedAttnParams& p, int r) {
  const int a = p.starts[r], b = p.starts[r + 1], kv = p.kv_len[r];
  PagedRequest x;
  x.q0 = min(max(a, 0), p.rows);
  x.n_new = min(max(b, x.q0), p.rows) - x.q0;
  if ((int64_t)x.n_new * p.group < p.least_rows || (int64_t)x.n_new * p.group > p.most_rows) x.n_new = 0;   // another launch's
  x.past = (int)max((int64_t)INT32_MIN / 2, (int64_t)kv - ((int64_t)b - a) + (x.q0 - (int64_t)a));
  x.keys = (int)min((int64_t)max(kv, 0), (int64_t)p.width * p.page.d);
  if (kv > x.keys && p.flag) atomicMax(p.flag, kPagedFlag);
  return x;
}

// Number of keys that new row i of the request sees.
__device__ __forceinline__ int visible_keys(const PagedRequest& x, int i) {
  return (int)min((int64_t)x.keys, max((int64_t)0, (int64_t)x.past + i + 1));
}

// Element offset of a request's key row (for one head, add head * sc.h); -1 on a page outside the pool.
__device__ __forceinline__ int64_t paged_row(const PagedAttnParams& p, const int32_t* table, int key) {
  const uint32_t at = p.page.div((uint32_t)key);
  const int page = table[at];
  if ((unsigned)page >= (unsigned)p.n_pages) {
    if (p.flag) atomicMax(p.flag, kPagedFlag);
    return -1;
  }
  return (int64_t)page * p.sc.b + (int64_t)(key - (int)at * (int)p.page.d) * p.sc.s;
}

// 16 bytes global -> shared (shared-window address); with bytes = 0 the destination is zeroed and nothing is read.
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Waits until at most N of this thread's groups of copies are in flight.
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace mt
