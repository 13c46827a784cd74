// Bookkeeping of the paged key/value cache on the GPU: block tables and slot maps from the requests'
// lengths, pages given back, new rows appended. No reference counterpart (mytorch_b200.h).
#include "paged.cuh"
#include "tempbuf.cuh"

namespace mt {

constexpr int kTabThreads = 1024;
constexpr int kMaxRequests = 8192;

__device__ __forceinline__ int clamp_i32(int64_t v) { return (int)min(v, (int64_t)INT32_MAX); }
__device__ __forceinline__ void paged_flag(int* flag) { if (flag) atomicMax(flag, kPagedFlag); }

// Exclusive prefix sums of two values per thread over the block; the totals go to all threads.
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t& total_a, int64_t& total_b) {
  __shared__ int64_t wa[32], wb[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
  int64_t ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ta = __shfl_up_sync(0xffffffffu, ia, o), tb = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) { ia += ta; ib += tb; }
  }
  if (lane == 31) { wa[warp] = ia; wb[warp] = ib; }
  __syncthreads();
  if (warp == 0) {
    int64_t sa = lane < warps ? wa[lane] : 0, sb = lane < warps ? wb[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t ta = __shfl_up_sync(0xffffffffu, sa, o), tb = __shfl_up_sync(0xffffffffu, sb, o);
      if (lane >= o) { sa += ta; sb += tb; }
    }
    wa[lane] = sa;
    wb[lane] = sb;
  }
  __syncthreads();
  total_a = wa[31];
  total_b = wb[31];
  a = ia - a + (warp ? wa[warp - 1] : 0);
  b = ib - b + (warp ? wb[warp - 1] : 0);
}

// The last r with prefix[r] <= x (prefix[0] = 0, non-decreasing, n entries).
__device__ __forceinline__ int find_request(const int* prefix, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// One launch for everything: a step of 64 requests is all latency. Every block scans all the lengths
// (two coalesced reads per request, L2 after the first block) into prefix sums in shared memory, so no
// block waits for another; block 0 writes what there is per request, and all blocks share the new
// table entries and the token rows, each found by a binary search in the prefix sums. Entries of this
// step's pages are computed from the list and never read back from the tables, which blocks write
// meanwhile. 64 requests with a token each 4.4 us, 1000 requests and 15598 tokens 6.5 (two round trips to memory, scans
// and a search).
__global__ void __launch_bounds__(kTabThreads)
paged_tables_kernel(const int32_t* __restrict__ held, const int32_t* __restrict__ fresh, int32_t* tables,
                    const int32_t* __restrict__ free_pages, const int32_t* __restrict__ n_free, int32_t* __restrict__ starts,
                    int32_t* __restrict__ kv_len, int32_t* __restrict__ position, int32_t* __restrict__ slot,
                    int32_t* __restrict__ n_free_out, int requests, int width, FastDiv page, int64_t list_len, int64_t rows,
                    int* flag) {
  extern __shared__ int tab_smem[];
  int* first_token = tab_smem;                   // [requests]
  int* first_new = tab_smem + requests;          // [requests]
  const int per = (requests + kTabThreads - 1) / kTabThreads;
  const int r0 = min(requests, (int)threadIdx.x * per), r1 = min(requests, r0 + per);
  auto pages_before = [&](int64_t h, int64_t kv, int& a, int& b) {     // new pages are [a, b)
    const int64_t d = page.d;
    a = (int)min((h + d - 1) / d, (int64_t)width);
    b = (int)min((kv + d - 1) / d, (int64_t)width);
  };
  int64_t tok = 0, pg = 0, tokens, pages;
  for (int r = r0; r < r1; ++r) {
    const int64_t h = max(held[r], 0), f = max(fresh[r], 0);
    int a, b;
    pages_before(h, h + f, a, b);
    tok += f;
    pg += b - a;
  }
  block_scan2(tok, pg, tokens, pages);
  for (int r = r0; r < r1; ++r) {
    const int64_t h = max(held[r], 0), f = max(fresh[r], 0);
    int a, b;
    pages_before(h, h + f, a, b);
    first_token[r] = clamp_i32(tok);
    first_new[r] = clamp_i32(pg);
    if (blockIdx.x == 0) {
      starts[r] = clamp_i32(tok);
      kv_len[r] = clamp_i32(h + f);
      if (h + f > (int64_t)width * page.d) paged_flag(flag);
    }
    tok += f;
    pg += b - a;
  }
  const int64_t have = min((int64_t)max(n_free[0], 0), list_len);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    starts[requests] = clamp_i32(tokens);
    n_free_out[0] = (int)max((int64_t)0, have - pages);
    if (pages > have || tokens > rows) paged_flag(flag);
  }
  __syncthreads();
  auto take = [&](int64_t k) { return k < have ? free_pages[have - 1 - k] : -1; };      // the step's k-th new page
  const int64_t stride = (int64_t)gridDim.x * kTabThreads, me = (int64_t)blockIdx.x * kTabThreads + threadIdx.x;
  for (int64_t e = me; e < pages; e += stride) {
    const int r = find_request(first_new, requests, (int)e);
    const int64_t h = max(held[r], 0);
    const int at = (int)((h + page.d - 1) / page.d) + (int)(e - first_new[r]);
    tables[(int64_t)r * width + at] = take(e);
  }
  for (int64_t i = me; i < rows; i += stride) {
    int pos = 0, where = -1;
    if (i < tokens) {
      const int r = find_request(first_token, requests, (int)i);
      const int64_t h = max(held[r], 0);
      const int64_t j = h + i - first_token[r];
      pos = clamp_i32(j);
      const int64_t at = j / page.d, first = (h + page.d - 1) / page.d;
      if (at < width) {
        const int id = at >= first ? take(first_new[r] + at - first) : tables[(int64_t)r * width + at];
        const int64_t s = (int64_t)id * page.d + (j - at * page.d);
        if (id >= 0 && s <= INT32_MAX) where = (int)s;
        else paged_flag(flag);
      }
    }
    position[i] = pos;
    slot[i] = where;
  }
}

// One block: warps count the pages of the requests that are done, the block turns the counts into places
// in the list, warps write. The order is that of requests and pages, whatever the scheduling. Bound by round trips to memory, several per
// request of a warp: 64 requests, 8 of them over with 128 pages each, 6 us; 1000, 100 over with 260 each, 20 us; 8192, all
// over at once with 64 each, 560 us.
__global__ void __launch_bounds__(kTabThreads)
paged_release_kernel(const int32_t* __restrict__ done, int32_t* tables, int32_t* kv_len, int32_t* free_pages, int32_t* n_free,
                     int requests, int width, FastDiv page, int64_t list_len, int* flag) {
  extern __shared__ int tab_smem[];              // [requests]: pages given back, then their first place
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = kTabThreads / 32;
  const int64_t have = min((int64_t)max(n_free[0], 0), list_len);
  auto pages_of = [&](int r) { return (int)min(((int64_t)max(kv_len[r], 0) + page.d - 1) / page.d, (int64_t)width); };
  for (int r = warp; r < requests; r += warps) {
    int n = 0;
    if (done[r])
      for (int j = lane, m = pages_of(r); j < m; j += 32) n += tables[(int64_t)r * width + j] >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) tab_smem[r] = n;
  }
  __syncthreads();
  const int per = (requests + kTabThreads - 1) / kTabThreads;
  const int r0 = min(requests, (int)threadIdx.x * per), r1 = min(requests, r0 + per);
  int64_t sum = 0, unused = 0, total, total_unused;
  for (int r = r0; r < r1; ++r) sum += tab_smem[r];
  block_scan2(sum, unused, total, total_unused);
  for (int r = r0; r < r1; ++r) { const int n = tab_smem[r]; tab_smem[r] = clamp_i32(sum); sum += n; }
  __syncthreads();
  for (int r = warp; r < requests; r += warps) {
    if (!done[r]) continue;
    const int m = pages_of(r);
    int64_t at = have + tab_smem[r];
    for (int j0 = 0; j0 < m; j0 += 32) {
      const int j = j0 + lane;
      const int id = j < m ? tables[(int64_t)r * width + j] : -1;
      const unsigned mask = __ballot_sync(0xffffffffu, id >= 0);
      const int64_t place = at + __popc(mask & ((1u << lane) - 1));
      if (id >= 0 && place < list_len) free_pages[place] = id;
      if (j < m) tables[(int64_t)r * width + j] = -1;
      at += __popc(mask);
    }
    __syncwarp();
    if (lane == 0) kv_len[r] = 0;
  }
  if (threadIdx.x == 0) {
    if (have + total > list_len) paged_flag(flag);
    n_free[0] = (int)min(have + total, list_len);
  }
}

// Copy rate bound. A thread moves 16-byte pieces (one element where something is not 16-byte aligned) of key rows and the
// same of the value rows, two at a time so that four loads are in flight; rows, heads and pieces come from 32-bit divisions
// by multiplication. 14225 tokens x 12 heads x 64 fp16: 13.0 us for 87 MB, a little above the copy rate as some of what it writes
// (44 MB) is still in L2 when it ends; 18.4 us from call to call.
template <typename V>
__global__ void __launch_bounds__(256)
paged_append_kernel(const V* __restrict__ k_new, const V* __restrict__ v_new, V* __restrict__ k_pages, V* __restrict__ v_pages,
                    mt_strides3 sk, mt_strides3 sv, mt_strides3 sc, const int32_t* __restrict__ slot, uint32_t total, FastDiv per_row,
                    FastDiv kv_heads, FastDiv page, int64_t n_slots, int* flag) {
  const uint32_t step = gridDim.x * 256u;
  for (uint32_t i0 = blockIdx.x * 256u + threadIdx.x; i0 < total; i0 += 2 * step) {
    V k[2], v[2];
    int64_t dst[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t i = i0 + u * step;                // below 2^31 + 2^21
      dst[u] = -1;
      if (i >= total) continue;
      const uint32_t r = per_row.div(i), c = i - r * per_row.d, row = kv_heads.div(r), h = r - row * kv_heads.d;
      const int s = slot[row];
      if (s < 0) continue;
      if (s >= n_slots) { paged_flag(flag); continue; }
      const uint32_t pg = page.div((uint32_t)s);
      dst[u] = (int64_t)pg * sc.b + (int64_t)h * sc.h + (int64_t)(s - pg * page.d) * sc.s + c;
      k[u] = k_new[row * sk.s + h * sk.h + c];
      v[u] = v_new[row * sv.s + h * sv.h + c];
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (dst[u] >= 0) { k_pages[dst[u]] = k[u]; v_pages[dst[u]] = v[u]; }
  }
}

template <typename V>
static int launch_append(const void* k_new, const void* v_new, void* k_pages, void* v_pages, mt_strides3 sk, mt_strides3 sv,
                         mt_strides3 sc, const int32_t* slot, int64_t rows, int64_t kv_heads, int64_t row_bytes, int elem,
                         int64_t page_size, int64_t n_pages, cudaStream_t st) {
  const int64_t per = (int64_t)sizeof(V) / elem, per_row = row_bytes / (int64_t)sizeof(V);
  auto in = [&](mt_strides3 s) { return mt_strides3{s.b / per, s.h / per, s.s / per}; };
  sk = in(sk); sv = in(sv); sc = in(sc);
  const int64_t at_once = ((1ll << 31) - 1) / (kv_heads * per_row);        // rows of a launch
  MT_REQUIRE(at_once >= 1, "paged_append: rows of all heads are limited to 2^31 pieces");
  for (int64_t r0 = 0; r0 < rows; r0 += at_once) {
    const int64_t n = rows - r0 < at_once ? rows - r0 : at_once, total = n * kv_heads * per_row;
    int64_t blocks = (total + 511) / 512;
    if (blocks > (int64_t)sm_count() * 32) blocks = (int64_t)sm_count() * 32;
    paged_append_kernel<V><<<(unsigned)blocks, 256, 0, st>>>(
        (const V*)k_new + r0 * sk.s, (const V*)v_new + r0 * sv.s, (V*)k_pages, (V*)v_pages, sk, sv, sc, slot + r0, (uint32_t)total,
        FastDiv((uint32_t)per_row), FastDiv((uint32_t)kv_heads), FastDiv((uint32_t)page_size), n_pages * page_size, device_flag_ptr());
    MT_LAUNCH_CHECK();
  }
  return MT_OK;
}

}  // namespace mt

using namespace mt;

extern "C" {

int mt_paged_tables(const int32_t* held, const int32_t* fresh, int32_t* tables, const int32_t* free_pages, const int32_t* n_free,
                    int32_t* starts, int32_t* kv_len, int32_t* position, int32_t* slot, int32_t* n_free_out, int64_t requests,
                    int64_t width, int64_t page_size, int64_t list_len, int64_t rows, void* stream) {
  MT_REQUIRE(held && fresh && tables && free_pages && n_free && starts && kv_len && position && slot && n_free_out,
             "paged_tables: bad arguments");
  MT_REQUIRE(requests >= 1 && requests <= kMaxRequests, "paged_tables: 1 to %d requests, got %lld", kMaxRequests, (long long)requests);
  MT_REQUIRE(width >= 1 && width < (1ll << 31) && page_size >= 1 && width * page_size < (1ll << 31) && page_size < (1ll << 30),
             "paged_tables: a table row has to span between 1 and 2^31 - 1 positions");
  MT_REQUIRE(list_len >= 0 && list_len < (1ll << 31) && rows >= 0 && rows < (1ll << 31), "paged_tables: bad sizes");
  MT_REQUIRE(kv_len != held && kv_len != fresh && n_free_out != n_free, "paged_tables: kv_len and n_free_out need buffers of their own");
  int64_t blocks = (rows + kTabThreads - 1) / kTabThreads;
  blocks = blocks < 1 ? 1 : blocks > sm_count() ? sm_count() : blocks;
  // raised whatever the size: the 48 KB that need no asking hold the static shared memory (512 bytes) as well
  static SmemLimit limit;
  if (int rc = limit.raise((const void*)paged_tables_kernel, 2 * kMaxRequests * (int)sizeof(int))) return rc;
  paged_tables_kernel<<<(unsigned)blocks, kTabThreads, 2 * requests * sizeof(int), as_stream(stream)>>>(
      held, fresh, tables, free_pages, n_free, starts, kv_len, position, slot, n_free_out, (int)requests, (int)width,
      FastDiv((uint32_t)page_size), list_len, rows, device_flag_ptr());
  MT_LAUNCH_CHECK();
  return MT_OK;
}

int mt_paged_release(const int32_t* done, int32_t* tables, int32_t* kv_len, int32_t* free_pages, int32_t* n_free, int64_t requests,
                     int64_t width, int64_t page_size, int64_t list_len, void* stream) {
  MT_REQUIRE(done && tables && kv_len && free_pages && n_free, "paged_release: bad arguments");
  MT_REQUIRE(requests >= 1 && requests <= kMaxRequests, "paged_release: 1 to %d requests, got %lld", kMaxRequests, (long long)requests);
  MT_REQUIRE(width >= 1 && width < (1ll << 31) && page_size >= 1 && width * page_size < (1ll << 31) && page_size < (1ll << 30) && list_len >= 0 && list_len < (1ll << 31),
             "paged_release: bad sizes");
  paged_release_kernel<<<1, kTabThreads, requests * sizeof(int), as_stream(stream)>>>(
      done, tables, kv_len, free_pages, n_free, (int)requests, (int)width, FastDiv((uint32_t)page_size), list_len, device_flag_ptr());
  MT_LAUNCH_CHECK();
  return MT_OK;
}

int mt_paged_append(const void* k_new, const void* v_new, void* k_pages, void* v_pages, mt_strides3 sk, mt_strides3 sv,
                    mt_strides3 spages, const int32_t* slot, int64_t rows, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                    int64_t n_pages, int dtype, void* stream) {
  MT_REQUIRE(k_new && v_new && k_pages && v_pages && slot && rows >= 0 && kv_heads > 0 && head_dim > 0 && n_pages >= 0,
             "paged_append: bad arguments");
  MT_REQUIRE(dtype == MT_F32 || dtype == MT_F16 || dtype == MT_BF16, "paged_append: unsupported dtype code %d", dtype);
  MT_REQUIRE(page_size >= 1 && page_size < (1ll << 30) && n_pages < (1ll << 31) && n_pages * page_size < (1ll << 31),
             "paged_append: a pool has to hold fewer than 2^31 rows");
  MT_REQUIRE(rows < (1ll << 31) && kv_heads < (1ll << 31) && head_dim < (1ll << 28), "paged_append: bad sizes");
  MT_REQUIRE(spages.b >= 0 && spages.h >= 0 && spages.s >= 0, "paged_append: negative strides of the pools");
  if (rows == 0) return MT_OK;
  const int e = (int)dtype_size(dtype);
  auto whole = [&](mt_strides3 s) { return s.h * e % 16 == 0 && s.s * e % 16 == 0; };
  const bool vec = head_dim * e % 16 == 0 && whole(sk) && whole(sv) && whole(spages) && spages.b * e % 16 == 0 && aligned16(k_new) &&
                   aligned16(v_new) && aligned16(k_pages) && aligned16(v_pages);
  cudaStream_t st = as_stream(stream);
  if (vec)
    return launch_append<uint4>(k_new, v_new, k_pages, v_pages, sk, sv, spages, slot, rows, kv_heads, head_dim * e, e, page_size, n_pages, st);
  if (e == 4)
    return launch_append<uint32_t>(k_new, v_new, k_pages, v_pages, sk, sv, spages, slot, rows, kv_heads, head_dim * e, e, page_size, n_pages, st);
  return launch_append<uint16_t>(k_new, v_new, k_pages, v_pages, sk, sv, spages, slot, rows, kv_heads, head_dim * e, e, page_size, n_pages, st);
}

}  // extern "C"
