// How attention over pages is shared out. Its work is a list of items - (request, key/value head, tile of
// M query rows), a row being a (new token, query head of the group) pair - and an item is a run of key
// tiles of KT keys. The host knows neither lengths nor how many items there are, and lengths differ
// by orders of magnitude, so every block finds its own share on the device: the items, each weighted with the
// keys its rows see, are laid end to end and cut into equal parts, one per block. A cut may fall inside an
// item, at a key tile; the blocks on both sides then leave partial results (unnormalised output, maximum
// and sum per row) that a second kernel joins in the order of the keys, so results do not depend on timing.
#pragma once
#include "paged.cuh"

namespace mt {

struct alignas(16) WorkPos { int r, hk, t, kt; };    // a key tile of an item; kt > 0: a cut inside the item

__device__ __forceinline__ bool same_item(const WorkPos& a, const WorkPos& b) { return a.r == b.r && a.hk == b.hk && a.t == b.t; }

template <int M>
__device__ __forceinline__ int row_tiles(const PagedAttnParams& p, const PagedRequest& x) {
  return (int)(((int64_t)x.n_new * p.group + M - 1) / M);
}

// Keys that the last row of tile t sees.
template <int M>
__device__ __forceinline__ int tile_keys(const PagedAttnParams& p, const PagedRequest& x, int t) {
  const int64_t rows = min((int64_t)(t + 1) * M, (int64_t)x.n_new * p.group);
  return visible_keys(x, (int)p.by_group.div((uint32_t)(rows - 1)));
}

// Key tiles that `keys` keys fill (up to 2^31 - 1 of them).
template <int KT>
__device__ __forceinline__ int key_tiles(int keys) { return (int)(((uint32_t)keys + KT - 1) / KT); }

// Weight of the first T of nt tiles of one head, in key tiles: increasing, in closed form and free of
// divisions (a block's first 2 us are this arithmetic, and every block does it). A tile's weight is FIXED for
// queries in and output out, and the keys that its rows see; `slope` is what a tile sees more than the one before, M / (group * KT), in
// units of 2^-16.
template <int KT, int FIXED>
__device__ __forceinline__ int64_t weight_upto(const PagedRequest& x, uint32_t slope, int T, int nt) {
  if (nt == 0) return 0;
  const int base = max(x.past, 0) / KT + FIXED, n = min(T, nt - 1);
  const int64_t w = (int64_t)n * base + (int64_t)(((uint64_t)((int64_t)n * (n + 1)) >> 1) * slope >> 16);
  return T < nt ? w : w + base + x.n_new / KT;
}

// Exclusive prefix sum of one value per thread and the block's total. `sh`: 33 values.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* sh, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
  int64_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += t;
  }
  if (lane == 31) sh[warp] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll 1
  for (int w = 0; w < warps; ++w) {
    if (w < warp) before += sh[w];
    total += sh[w];
  }
  return s - v + before;
}

struct WorkShare { WorkPos begin; const WorkPos* end; int blocks; };    // blocks that have work

// This block's share (valid until the block ends: `end` is in shared memory); every thread calls it and gets
// the same answer (`blocks`: thread 0). `least`: at least so many key tiles per block, fixed costs included. Cuts nearer
// to an item's ends than 1/NEAR of a share move there; with `whole` all do, and no item is cut. Warp 0 finds where the share
// begins and warp 1 where it ends, each with prefix sums of its own over up to 256 requests (two round trips to memory and 3000
// cycles less than sums over the block first, which longer lists take).
template <int M, int KT, int FIXED, int NEAR>
__device__ __forceinline__ WorkShare find_share(const PagedAttnParams& p, int least, uint32_t slope, bool whole) {
  __shared__ int64_t sums[33];
  __shared__ int64_t before[2];          // of the two cuts: weights before the thread's requests
  __shared__ int owner[2];
  __shared__ WorkPos found[2];
  const int lane = threadIdx.x & 31, e = threadIdx.x >> 5;
  auto weights = [&](int r0, int r1) {
    int64_t w = 0;
#pragma unroll 2
    for (int r = r0; r < r1; ++r) {
      const PagedRequest x = paged_request(p, r);
      const int nt = row_tiles<M>(p, x);
      w += weight_upto<KT, FIXED>(x, slope, nt, nt) * p.kv_heads;
    }
    return w;
  };
  // Every block computes the same numbers, and rounding keeps the order of the cuts: that is all they need.
  auto blocks_of = [&](int64_t total) { return (int)fmaxf(1.f, fminf((float)gridDim.x, (float)total / (float)least)); };
  auto cut_of = [&](int64_t total, int blocks, int c) { return (int64_t)((float)total * ((float)c / (float)blocks)); };
  const bool few = p.requests <= 256;
  int64_t total = 0, cut = 0;
  int blocks = 0, first = -1;            // first: where the search for the cut starts, in the thread that makes it
  if (few) {
    if (e < 2) {
      const int per = (p.requests + 31) / 32, r0 = min(p.requests, lane * per);
      const int64_t mine = weights(r0, min(p.requests, r0 + per));
      int64_t at = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at += t;
      }
      total = __shfl_sync(0xffffffffu, at, 31);
      at -= mine;
      blocks = blocks_of(total);
      const int c = (int)blockIdx.x + e;
      cut = cut_of(total, blocks, c) - at;
      if (c < blocks && cut >= 0 && cut < mine) first = r0;
    }
  } else {
    const int per = (p.requests + (int)blockDim.x - 1) / (int)blockDim.x;
    const int r0 = min(p.requests, (int)threadIdx.x * per);
    const int64_t mine = weights(r0, min(p.requests, r0 + per));
    if (threadIdx.x < 2) owner[threadIdx.x] = -1;
    const int64_t at = block_scan(mine, sums, total);
    blocks = blocks_of(total);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = (int)blockIdx.x + k;
      const int64_t x = cut_of(total, blocks, c);
      if (c < blocks && x >= at && x < at + mine) { before[k] = at; owner[k] = r0; }
    }
    __syncthreads();
    if (e < 2 && lane == 0 && owner[e] >= 0) {
      first = owner[e];
      cut = cut_of(total, blocks, (int)blockIdx.x + e) - before[e];
    }
  }
  if (e < 2) {
    if (first >= 0) {
      int64_t head = 0;
      PagedRequest x{};
      WorkPos f;
      int nt = 0;
#pragma unroll 1
      for (f.r = first;; ++f.r) {
        x = paged_request(p, f.r);
        nt = row_tiles<M>(p, x);
        head = weight_upto<KT, FIXED>(x, slope, nt, nt);
        if (cut < head * p.kv_heads) break;
        cut -= head * p.kv_heads;
      }
      f.hk = (int)__fdividef((float)cut, (float)head);
      cut -= f.hk * head;
#pragma unroll 1
      for (; cut < 0; cut += head) --f.hk;
#pragma unroll 1
      for (; cut >= head; cut -= head) ++f.hk;
      int lo = 0, hi = nt;                           // the last tile that begins at or before the cut
#pragma unroll 1
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (weight_upto<KT, FIXED>(x, slope, mid, nt) <= cut) lo = mid; else hi = mid;
      }
      const int64_t begin = weight_upto<KT, FIXED>(x, slope, lo, nt), width = weight_upto<KT, FIXED>(x, slope, lo + 1, nt) - begin;
      const int n = key_tiles<KT>(tile_keys<M>(p, x, lo));
      const int kt = min(n - 1, (int)((float)(cut - begin) * (float)n / (float)width));
      const int snap = whole ? n / 2 : (int)fminf(1e9f, (float)total / (float)(NEAR * blocks));
      f.t = lo;
      f.kt = kt <= snap ? 0 : kt;
      if (f.kt && (whole || n - kt <= snap)) { ++f.t; f.kt = 0; }
      found[e] = f;
    }
    if (__ballot_sync(0xffffffffu, first >= 0) == 0 && lane == 0) found[e] = WorkPos{p.requests, 0, 0, 0};   // the list's end
  }
  __syncthreads();
  return WorkShare{found[0], &found[1], blocks};     // without a share both are the list's end
}

template <int M, int KT>
inline uint32_t tile_slope(int group) { return (uint32_t)(((uint64_t)M << 16) / ((uint64_t)group * KT)); }

struct WorkItem {
  int r, hk, t;
  int k0, k1, n;                         // key tiles [k0, k1) of n
  int rows;                              // of the tile
  int keys;                              // that its last row sees
  PagedRequest x;
};

// Walks a share item by item.
template <int M, int KT>
struct WorkIter {
  WorkPos cur;
  const WorkPos* last;
  int loaded, nt;
  PagedRequest x;
  __device__ __forceinline__ void start(const WorkShare& s) { cur = s.begin; last = s.end; loaded = -1; nt = 0; }
  __device__ __forceinline__ bool next(const PagedAttnParams& p, WorkItem& it) {
    const WorkPos end = *last;
#pragma unroll 1
    for (;;) {
      if (cur.r >= p.requests) return false;
      if (cur.r > end.r || (cur.r == end.r && (cur.hk > end.hk || (cur.hk == end.hk && (cur.t > end.t || (cur.t == end.t && cur.kt >= end.kt))))))
        return false;
      if (loaded != cur.r) {
        x = paged_request(p, cur.r);
        nt = row_tiles<M>(p, x);
        loaded = cur.r;
      }
      if (cur.t < nt) break;
      cur.t = cur.kt = 0;
      if (nt == 0 || ++cur.hk == p.kv_heads) { cur.hk = 0; ++cur.r; }
    }
    it.r = cur.r; it.hk = cur.hk; it.t = cur.t; it.x = x;
    it.rows = (int)min((int64_t)M, (int64_t)x.n_new * p.group - (int64_t)cur.t * M);
    it.keys = tile_keys<M>(p, x, cur.t);
    it.n = key_tiles<KT>(it.keys);
    it.k0 = cur.kt;
    it.k1 = same_item(cur, end) ? min(end.kt, it.n) : it.n;
    ++cur.t;
    cur.kt = 0;
    return true;
  }
};

// Partial results of a block's first and last item, where a cut runs through them: [2 per block][M rows]
// of D sums (laid out by partial_row), then the rows' maxima (log2 domain) and weights' sums; `cuts`: where every block begins, the number of
// blocks with work behind the last.
struct WorkPartials {
  float* o;
  float* ml;
  WorkPos* cuts;
};

// Where the tensor-core kernel (256 rows) keeps 32 rows' columns [col, col + 32) of a partial result, in floats from
// the start: 32 rows of 128 bytes, whose 16-byte pieces lie swizzled by row as its staging buffers have them.
template <int D>
__device__ __forceinline__ int64_t partial_at(int slot, int row, int col) {
  return (((int64_t)slot * 8 + row / 32) * (D / 32) + col / 32) * 1024;
}
// E neighbouring columns of a row of a partial result.
template <int D, int M, int E>
__device__ __forceinline__ int64_t partial_row(int slot, int row, int col) {
  if (M < 256) return ((int64_t)slot * M + row) * D + col;
  return partial_at<D>(slot, row, col) + (row & 31) * 32 + ((((col & 31) >> 2) ^ (row & 7)) << 2) + (col & 3);
}

__device__ __forceinline__ int partial_slot(const WorkItem& it) {
  return it.k0 > 0 ? 2 * (int)blockIdx.x : it.k1 < it.n ? 2 * (int)blockIdx.x + 1 : -1;
}

inline size_t partial_bytes(int blocks, int M, int D) {
  return (size_t)blocks * 2 * M * (D + 2) * sizeof(float) + (size_t)(blocks + 1) * sizeof(WorkPos);
}
inline WorkPartials partials_in(void* buf, int blocks, int M, int D) {
  WorkPartials w;
  w.o = (float*)buf;
  w.ml = w.o + (size_t)blocks * 2 * M * D;
  w.cuts = (WorkPos*)(w.ml + (size_t)blocks * 2 * M * 2);
  return w;
}

// The block whose share begins at blockIdx.x tells the joining kernel so, if there is one.
__device__ __forceinline__ void publish_share(const WorkShare& s, const WorkPartials& w) {
  if (threadIdx.x == 0 && w.cuts) {
    w.cuts[blockIdx.x] = s.begin;
    if (blockIdx.x == 0) w.cuts[gridDim.x] = WorkPos{s.blocks, 0, 0, 0};
  }
}

// Token and query head of row `row` of an item's tile.
template <int M>
__device__ __forceinline__ void row_of(const PagedAttnParams& p, const WorkItem& it, int row, int& token, int& head) {
  const uint32_t at = (uint32_t)it.t * M + row;
  token = (int)p.by_group.div(at);
  head = it.hk * p.group + (int)(at - (uint32_t)token * p.group);
}

// Lane l's D/32 neighbouring elements of an output row.
template <typename T, int E>
__device__ __forceinline__ void store_row(const PagedAttnParams& p, const PagedRequest& x, int token, int head, const float (&v)[E]) {
  T* op = (T*)p.o + (int64_t)(x.q0 + token) * p.so.s + (int64_t)head * p.so.h + (threadIdx.x & 31) * E;
  if (p.o_quads) {
    struct alignas(sizeof(T) * E) Pack { T t[E]; } pack;
#pragma unroll
    for (int e = 0; e < E; ++e) pack.t[e] = from_f<T>(v[e]);
    *reinterpret_cast<Pack*>(op) = pack;
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) op[e] = from_f<T>(v[e]);
  }
}

// One output row (a token's head) by one warp, straight from the definition: lane l holds D/32
// neighbouring elements of q and o, scores are fp32 dot products, and only the visible keys are touched.
// The tiled kernels' masks are weights of zero, which a value that is not finite turns into NaN; rows
// that come out as NaN are therefore computed again here.
template <typename T, int D>
__device__ __noinline__ void paged_row_plain(const PagedAttnParams& p, PagedRequest x, int r, int i, int h) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t head = (int64_t)(h / p.group) * p.sc.h;
  const T* kp = (const T*)p.kp + head + lane * E;
  const T* vp = (const T*)p.vp + head + lane * E;
  const T* qp = (const T*)p.q + (int64_t)(x.q0 + i) * p.sq.s + (int64_t)h * p.sq.h + lane * E;
  const int32_t* table = p.tables + (int64_t)r * p.width;
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) { q[e] = to_f(qp[e]) * p.scale_log2; o[e] = 0.f; }
  const int n = visible_keys(x, i);
#pragma unroll 1
  for (int j = 0; j < n; ++j) {
    const int64_t at = paged_row(p, table, j);
    if (at < 0) continue;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s = fmaf(q[e], to_f(kp[at + e]), s);
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    if (mn == -INFINITY && !isnan(s)) continue;      // no finite score yet
    const float c = m == -INFINITY ? 0.f : exp2f(m - mn), w = exp2f(s - (mn == -INFINITY ? 0.f : mn));
    m = mn;
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(w, to_f(vp[at + e]), o[e] * c);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = l == 0.f ? 0.f : o[e] / l;
  store_row<T, E>(p, x, i, h, o);
}

// Joins the partial results of the items that cuts run through: block (c, y) takes the item whose first cut
// is the one between blocks c and c + 1. A lane looks one piece up, so that a row of up to
// 32 pieces costs four round trips to L2 whatever their number (8 us for seven pieces looked up one after the other,
// 2.5 so); the pieces are added in the order of the keys.
template <typename T, int D, int M, int KT>
__global__ void __launch_bounds__(128)
paged_join_kernel(const __grid_constant__ PagedAttnParams p, const WorkPartials w, int grid) {
  constexpr int E = D / 32;
  grid_dependency_wait();
  allow_dependents();
  const int blocks = w.cuts[grid].r, c = (int)blockIdx.x + 1;
  const WorkPos cut = w.cuts[c], before = w.cuts[c - 1];
  if (c >= blocks || cut.kt == 0 || (before.kt > 0 && same_item(before, cut))) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  WorkItem it;
  it.r = cut.r; it.hk = cut.hk; it.t = cut.t;
  it.x = paged_request(p, cut.r);
  it.rows = (int)min((int64_t)M, (int64_t)it.x.n_new * p.group - (int64_t)cut.t * M);
  int last = c;                                      // the item's pieces: slot 2c-1, then slots 2j of blocks c..last
#pragma unroll 1
  for (;;) {
    const int j = last + 1 + lane;
    const bool inside = j < blocks && same_item(w.cuts[j], cut) && w.cuts[j].kt > 0;
    const uint32_t out = __ballot_sync(0xffffffffu, !inside);
    if (out) { last += __ffs((int)out) - 1; break; }
    last += 32;
  }
  const int pieces = last - c + 2;
  // W rows of a warp go side by side, so that their lookups and loads overlap (four rows one after the other: 13 us
  // for 100 items of 256 rows in two or three pieces).
  constexpr int W = M >= 64 ? 4 : 1;
  const int first = ((int)blockIdx.y * 4 + warp) * W;
  if (first >= it.rows) return;
  float m[W], l[W], o[W][E];
#pragma unroll
  for (int k = 0; k < W; ++k) {
    m[k] = -INFINITY;
    l[k] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) o[k][e] = 0.f;
  }
#pragma unroll 1
  for (int i0 = 0; i0 < pieces; i0 += 32) {
    const int i = i0 + lane, j = c + i - 1;
    int slot = i < pieces ? (i == 0 ? 2 * c - 1 : 2 * j) : -1;
    if (slot >= 0 && i > 0 && j < last && w.cuts[j + 1].kt == w.cuts[j].kt) slot = -1;   // two cuts at one key tile: nothing was written
    float2 ml[W];
    float a[W];
#pragma unroll
    for (int k = 0; k < W; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      if (slot >= 0) ml[k] = *reinterpret_cast<const float2*>(w.ml + ((int64_t)slot * M + first + k) * 2);
    }
#pragma unroll
    for (int k = 0; k < W; ++k) {
      const float mn = fmaxf(m[k], warp_max(ml[k].x));
      // without a maximum there are no weights, or only NaN ones, which stay
      const float keep = m[k] == -INFINITY ? 0.f : exp2f(m[k] - mn);
      a[k] = ml[k].x == -INFINITY ? (isnan(ml[k].y) ? ml[k].y : 0.f) : exp2f(ml[k].x - mn);
      m[k] = mn;
      l[k] = l[k] * keep + warp_sum(slot >= 0 && first + k < it.rows ? ml[k].y * a[k] : 0.f);
#pragma unroll
      for (int e = 0; e < E; ++e) o[k][e] *= keep;
    }
    const int n = min(32, pieces - i0);
#pragma unroll W == 1 ? 8 : 2
    for (int q = 0; q < n; ++q) {
      const int s = __shfl_sync(0xffffffffu, slot, q);
      struct alignas(4 * E) Pack { float t[E]; } v[W];
#pragma unroll
      for (int k = 0; k < W; ++k) {
        v[k] = Pack{};
        if (s >= 0) v[k] = *reinterpret_cast<const Pack*>(w.o + partial_row<D, M, E>(s, first + k, lane * E));
      }
#pragma unroll
      for (int k = 0; k < W; ++k) {
        const float f = __shfl_sync(0xffffffffu, a[k], q);
#pragma unroll
        for (int e = 0; e < E; ++e) o[k][e] = fmaf(v[k].t[e], f, o[k][e]);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if (first + k >= it.rows) break;
    int token, head;
    row_of<M>(p, it, first + k, token, head);
    bool nan = false;
    const float inv = l[k] == 0.f ? 0.f : 1.f / l[k];
#pragma unroll
    for (int e = 0; e < E; ++e) { o[k][e] *= inv; nan |= isnan(o[k][e]); }
    if (__any_sync(0xffffffffu, nan)) paged_row_plain<T, D>(p, it.x, it.r, token, head);
    else store_row<T, E>(p, it.x, token, head, o[k]);
  }
}

template <typename T, int D, int M, int KT>
static int launch_join(const PagedAttnParams& p, const WorkPartials& w, int grid, cudaStream_t st) {
  if (grid < 2) return MT_OK;
  MT_CHECK_CUDA(launch_overlapped(paged_join_kernel<T, D, M, KT>, dim3((unsigned)grid - 1, M >= 64 ? M / 16 : (M + 3) / 4), dim3(128), 0, st, p, w, grid));
  count_launch();
  return MT_OK;
}

}  // namespace mt
