// Attention over pages for few query rows per key/value head: decoding steps and a few drafted tokens.
//
// HBM bound: every key and value row of a head is read once (2 D bytes a key in half precision, against
// 4 D operations per query row). A block of four warps works on one item at a time: M rows (tokens times the
// query heads of the group) and a run of key tiles. A warp owns a part of each tile (16 or 32 keys, 8 in fp32)
// and has a ring of stages of its own, filled by 16-byte cp.async: page lookups run one tile ahead of the loads,
// loads one tile ahead of the products (two in fp32, except for 8 rows of 128) and on across item boundaries, and no warp waits for
// another until an item's end. Rows that are not there (behind the last key, on a bad page) are
// filled with zeros and masked, so whatever lies in unused rows of a page is never read.
// 256 x 12 heads x 128..1000 keys x 64 fp16: 84 us, 5.1 TB/s (77 % of the copy rate); 32 x 10/2 heads x 300..2000 x 128 bf16: 20 us, of
// which the keys and values need 6 (finding shares, first loads, joining and launches the rest).
//   half: transposed products by mma.sync (m16n8k16), S^T = K Q^T and O^T += V^T P^T, so that the keys fill
//         the 16 rows of an MMA and the queries are its 8 columns: with one to eight rows per item (decoding) half the products,
//         registers and exponentials of the other way round. P^T moves from accumulators to operands by
//         movmatrix, as a pair of halves (rounded value and remainder): the tensor pipe has room, the weights
//         keep about fp32's precision, and the output is as exact as one rounding allows.
//   fp32: lane = key and quarter of head_dim for the scores, lane = elements of head_dim for the output.
// The online softmax is kept per warp; warps join at an item's end through shared memory, blocks through
// the partial results of paged_work.cuh.
#include "attention_paged.cuh"
#include "paged_work.cuh"
#include "tempbuf.cuh"

namespace mt {

constexpr int kFewWarps = 4;

// M rows per item: 8 or 16 in half precision, 1, 2, 4 or 8 in fp32.
template <typename T, int D, int M> struct FewCfg {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kRows = kHalf ? (D == 64 ? 32 : 16) : 8;  // keys of a warp in a tile
  static constexpr int KT = kRows * kFewWarps;
  static constexpr int kChunks = D * (int)sizeof(T) / 16;        // 16-byte pieces of a row
  static constexpr int kTile = kRows * kChunks * 16;             // bytes of a warp's keys (or values) of one tile
  static constexpr int kStages = kHalf ? 2 : M == 8 && D == 128 ? 2 : 3;
  static constexpr int kRing = kStages * 2 * kTile;              // per warp
  static constexpr int kPitch = D + 4;                           // of a row of results in shared memory, floats
  static constexpr int kParts = kHalf ? 2 : kFewWarps;           // results that meet there
  static constexpr int kOffMerge = kFewWarps * kRing;
  static constexpr int kOffQ = kOffMerge + kParts * M * kPitch * 4;   // fp32: the scaled queries
  static constexpr int kOffStat = kOffQ + (kHalf ? 0 : M * D * 4);    // maxima and sums, [2][warps][M]
  static constexpr int kSmem = kOffStat + kFewWarps * M * 2 * 4 + kFewWarps * kStages * 4;
  // 228 KB per SM, of which every block costs 1 KB and 336 bytes of static shared memory besides its own
  static constexpr int kFit = 233472 / (kSmem + 1024 + 336);
  static constexpr int kBlocks = kFit < (kHalf ? 3 : 4) ? kFit : (kHalf ? 3 : 4);
  static_assert(kBlocks >= 2, "two blocks per SM");
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__half>(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16<__nv_bfloat16>(float (&c)[4], const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transposes an 8x8 matrix of halves held as one pair per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T> __device__ __forceinline__ uint32_t pair_bits(T a, T b) {
  return (uint32_t)*reinterpret_cast<uint16_t*>(&a) | (uint32_t)*reinterpret_cast<uint16_t*>(&b) << 16;
}

// A warp's ring of key and value tiles: the load side of the pipeline. The warp holds 32 neighbouring entries of the
// request's table, one per lane; a new window is asked for when the next tile is not in it, while the
// tile before is on its way.
template <typename T, int D, int M>
struct FewLoader {
  using Cfg = FewCfg<T, D, M>;
  WorkIter<M, Cfg::KT> iter;
  WorkItem it;
  bool valid;
  int kt, window, page;                  // window: first table entry held, -1: none; page: lane's entry
  uint32_t ring;
  uint32_t* masks;                       // [stages]: which of the tile's rows are there

  __device__ __forceinline__ int first_key(int warp) const { return kt * Cfg::KT + warp * Cfg::kRows; }
  __device__ __forceinline__ void advance(const PagedAttnParams& p, int warp, int lane) {
#pragma unroll 1
    while (valid && kt >= it.k1) {
      valid = iter.next(p, it);
      if (valid) { kt = it.k0; window = -1; }
    }
    if (!valid) return;
    const int key0 = first_key(warp), n = min(Cfg::kRows, it.keys - key0);
    if (n <= 0) return;                                          // no row of this warp's in the tile
    const int a = (int)p.page.div((uint32_t)key0), b = (int)p.page.div((uint32_t)(key0 + n - 1));
    if (window >= 0 && b - window < 32) return;
    window = a;
    page = lane < p.width - a ? p.tables[(int64_t)it.r * p.width + a + lane] : -1;
  }
  __device__ __forceinline__ void start(const PagedAttnParams& p, const WorkShare& s, int warp, int lane) {
    iter.start(s);
    it.k1 = 0;
    kt = 0;
    window = -1;
    valid = true;
    advance(p, warp, lane);
  }
  // Queues the loads of the tile under the cursor into `stage`, one commit group per call.
  __device__ __forceinline__ void issue(const PagedAttnParams& p, int stage, int warp, int lane) {
    if (valid) {
      const int key = first_key(warp) + (lane % Cfg::kRows);
      const uint32_t at = p.page.div((uint32_t)key);
      const int id = __shfl_sync(0xffffffffu, page, (int)at - window);       // lanes behind the last key read anything
      int64_t off = -1;
      if (key < it.keys) {
        if ((unsigned)id < (unsigned)p.n_pages)
          off = (int64_t)id * p.sc.b + (int64_t)(key - (int)(at * p.page.d)) * p.sc.s + (int64_t)it.hk * p.sc.h;
        else if (p.flag) atomicMax(p.flag, kPagedFlag);
      }
      const uint32_t mask = __ballot_sync(0xffffffffu, off >= 0) & (uint32_t)((1ull << Cfg::kRows) - 1);
      if (lane == 0) masks[stage] = mask;
      if (mask) {
        const uint32_t kd = ring + stage * 2 * Cfg::kTile, vd = kd + Cfg::kTile;
#pragma unroll
        for (int i = 0; i < Cfg::kRows * Cfg::kChunks / 32; ++i) {
          const int row = (i * 32 + lane) / Cfg::kChunks, c = (i * 32 + lane) % Cfg::kChunks;
          const int64_t o = __shfl_sync(0xffffffffu, off, row);
          const uint32_t to = (row * Cfg::kChunks + (c ^ (row & 7))) * 16;
          const int64_t src = o >= 0 ? o + c * (16 / (int)sizeof(T)) : 0;
          copy16_async(kd + to, (const T*)p.kp + src, o >= 0 ? 16 : 0);
          copy16_async(vd + to, (const T*)p.vp + src, o >= 0 ? 16 : 0);
        }
      }
      ++kt;
      advance(p, warp, lane);
    }
    copy_commit();
  }
};

// An item's results, from `Cfg::kParts` parts in shared memory, weighted by `factor(part, row)`: to the output, or to
// the block's partial results. top, sum: of a row.
template <typename T, int D, int M, typename Cfg, typename Row, typename Factor>
__device__ __forceinline__ void few_finish(const PagedAttnParams& p, const WorkPartials& w, const WorkItem& it, const float* merge,
                                           Row row_stats, Factor factor) {
  constexpr int E = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = partial_slot(it);
#pragma unroll 1
  for (int g = warp; g < it.rows; g += kFewWarps) {
    float top, sum, o[E];
    row_stats(g, top, sum);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
    for (int v = 0; v < Cfg::kParts; ++v) {
      const float f = factor(v, g, top);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = fmaf(merge[(v * M + g) * Cfg::kPitch + lane * E + e], f, o[e]);
    }
    if (slot >= 0) {
      struct alignas(4 * E) Pack { float t[E]; } pack;
#pragma unroll
      for (int e = 0; e < E; ++e) pack.t[e] = o[e];
      *reinterpret_cast<Pack*>(w.o + ((int64_t)slot * M + g) * D + lane * E) = pack;
      if (lane == 0) *reinterpret_cast<float2*>(w.ml + ((int64_t)slot * M + g) * 2) = make_float2(top, sum);
      continue;
    }
    int token, head;
    row_of<M>(p, it, g, token, head);
    bool nan = false;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int e = 0; e < E; ++e) { o[e] *= inv; nan |= isnan(o[e]); }
    if (__any_sync(0xffffffffu, nan)) paged_row_plain<T, D>(p, it.x, it.r, token, head);
    else store_row<T, E>(p, it.x, token, head, o);
  }
}

// The weight of a part with maximum m and sum l where the maximum of all is `top`. Without a maximum there are no
// weights, or only NaN ones, which stay.
__device__ __forceinline__ float part_weight(float m, float l, float top) {
  return m == -INFINITY ? (isnan(l) ? l : 0.f) : exp2f(m - top);
}

template <typename T, int D, int M>
__global__ void __launch_bounds__(kFewWarps * 32, FewCfg<T, D, M>::kBlocks)
paged_few_half_kernel(const __grid_constant__ PagedAttnParams p, const WorkPartials w, int least, uint32_t slope, int whole) {
  using Cfg = FewCfg<T, D, M>;
  constexpr int NT = M / 8, KM = Cfg::kRows / 16, C = Cfg::kChunks;
  extern __shared__ __align__(128) uint8_t few_smem[];
  float* merge = reinterpret_cast<float*>(few_smem + Cfg::kOffMerge);
  float* stat = reinterpret_cast<float*>(few_smem + Cfg::kOffStat);            // [warps][M] maxima, then sums
  uint32_t* masks = reinterpret_cast<uint32_t*>(stat + kFewWarps * M * 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  allow_dependents();
  const WorkShare share = find_share<M, Cfg::KT, 1, 8>(p, least, slope, whole);
  publish_share(share, w);
  FewLoader<T, D, M> load;
  load.ring = smem_addr(few_smem) + warp * Cfg::kRing;
  load.masks = masks + warp * Cfg::kStages;
  load.start(p, share, warp, lane);
#pragma unroll 1
  for (int s = 0; s < Cfg::kStages; ++s) load.issue(p, s, warp, lane);
  WorkIter<M, Cfg::KT> iter;
  iter.start(share);
  WorkItem it;
  int stage = 0;
  const int quad = lane >> 2, pair = 2 * (lane & 3);     // a fragment's row (or column), and its first element along the other side
  while (iter.next(p, it)) {
    uint32_t qf[NT][D / 16][2];                          // Q^T as the right operand: column = query row
    int tok, head;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = 8 * n + quad;
      row_of<M>(p, it, row, tok, head);
      const bool real = row < it.rows;
      const T* q = (const T*)p.q + (real ? (int64_t)(it.x.q0 + tok) * p.sq.s + (int64_t)head * p.sq.h + pair : 0);
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const T* at = q + k * 16 + h * 8;
          qf[n][k][h] = !real ? 0u : p.q_pairs ? *reinterpret_cast<const uint32_t*>(at) : pair_bits(at[0], at[1]);
        }
    }
    row_of<M>(p, it, 0, tok, head);
    const int first_lim = visible_keys(it.x, tok);       // the tile's first row sees the fewest keys
    float acc[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) acc[n][d][0] = acc[n][d][1] = acc[n][d][2] = acc[n][d][3] = 0.f;
    }
#pragma unroll 1
    for (int kt = it.k0; kt < it.k1; ++kt) {
      copy_wait<Cfg::kStages - 1>();
      __syncwarp();
      const uint32_t mask = load.masks[stage];
      const int key0 = kt * Cfg::KT + warp * Cfg::kRows;
      if (mask) {
        const uint32_t kb = load.ring + stage * 2 * Cfg::kTile, vb = kb + Cfg::kTile;
        float s[KM][NT][4];
#pragma unroll
        for (int i = 0; i < KM; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n) s[i][n][0] = s[i][n][1] = s[i][n][2] = s[i][n][3] = 0.f;
        {
          const int row = lane & 15, half = lane >> 4;
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int i = 0; i < KM; ++i) {
              uint32_t a[4];
              ldm4(a, kb + ((16 * i + row) * C + ((2 * k + half) ^ (row & 7))) * 16);
#pragma unroll
              for (int n = 0; n < NT; ++n) mma16<T>(s[i][n], a, qf[n][k][0], qf[n][k][1]);
            }
        }
        const bool full = mask == (uint32_t)((1ull << Cfg::kRows) - 1) && key0 <= first_lim - Cfg::kRows;
        if (!full) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = 8 * n + pair + e;
              row_of<M>(p, it, row, tok, head);
              const int lim = row < it.rows ? visible_keys(it.x, tok) : 0;
#pragma unroll
              for (int i = 0; i < KM; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int j = 16 * i + 8 * h + quad;
                  if (!((mask >> j) & 1) || key0 + j >= lim) s[i][n][2 * h + e] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float x[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < KM; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int e = 0; e < 2; ++e) x[e] = fmaxf(x[e], s[i][n][2 * h + e]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            x[0] = fmaxf(x[0], __shfl_xor_sync(0xffffffffu, x[0], o));
            x[1] = fmaxf(x[1], __shfl_xor_sync(0xffffffffu, x[1], o));
          }
          x[0] = fmaxf(x[0] * p.scale_log2, m[n][0]);
          x[1] = fmaxf(x[1] * p.scale_log2, m[n][1]);
          if (__any_sync(0xffffffffu, x[0] > m[n][0] || x[1] > m[n][1])) {
            const float c0 = m[n][0] == -INFINITY ? 0.f : exp2f(m[n][0] - x[0]), c1 = m[n][1] == -INFINITY ? 0.f : exp2f(m[n][1] - x[1]);
            m[n][0] = x[0];
            m[n][1] = x[1];
            l[n][0] *= c0;
            l[n][1] *= c1;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) { acc[n][d][0] *= c0; acc[n][d][1] *= c1; acc[n][d][2] *= c0; acc[n][d][3] *= c1; }
          }
          const float u0 = m[n][0] == -INFINITY ? 0.f : m[n][0], u1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
          uint32_t hi[KM][2], lo[KM][2];                 // P^T as the right operand
#pragma unroll
          for (int i = 0; i < KM; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float p0 = exp2f(fmaf(s[i][n][2 * h], p.scale_log2, -u0)), p1 = exp2f(fmaf(s[i][n][2 * h + 1], p.scale_log2, -u1));
              l[n][0] += p0;
              l[n][1] += p1;
              const T h0 = from_f<T>(p0), h1 = from_f<T>(p1);
              hi[i][h] = transpose8(pair_bits(h0, h1));
              lo[i][h] = transpose8(pair_bits(from_f<T>(p0 - to_f(h0)), from_f<T>(p1 - to_f(h1))));
            }
          const int row = (lane & 7) + ((lane >> 4) << 3), next = (lane >> 3) & 1;
#pragma unroll
          for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int i = 0; i < KM; ++i) {
              uint32_t a[4];
              ldm4t(a, vb + ((16 * i + row) * C + ((2 * d + next) ^ (row & 7))) * 16);
              mma16<T>(acc[n][d], a, hi[i][0], hi[i][1]);
              mma16<T>(acc[n][d], a, lo[i][0], lo[i][1]);
            }
        }
      }
      __syncwarp();
      load.issue(p, stage, warp, lane);
      stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;
    }
    // the warps' results: a common maximum, then warps 2 and 3 into 0 and 1, and those two in few_finish
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
        if (quad == 0) {
          stat[warp * M + 8 * n + pair + e] = m[n][e];
          stat[(kFewWarps + warp) * M + 8 * n + pair + e] = l[n][e];
        }
      }
    __syncthreads();
    auto row_stats = [&](int g, float& top, float& sum) {
      top = -INFINITY;
      sum = 0.f;
#pragma unroll
      for (int v = 0; v < kFewWarps; ++v) top = fmaxf(top, stat[v * M + g]);
#pragma unroll
      for (int v = 0; v < kFewWarps; ++v) {
        const float lv = stat[(kFewWarps + v) * M + g];
        sum = fmaf(lv, part_weight(stat[v * M + g], lv, top), sum);
      }
    };
    auto part = [&](int v, int n, int d, int i) -> float& {   // element i of a fragment in part v
      return merge[(v * M + 8 * n + pair + (i & 1)) * Cfg::kPitch + 16 * d + 8 * (i >> 1) + quad];
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top, sum;
        row_stats(8 * n + pair + e, top, sum);
        f[e] = part_weight(m[n][e], l[n][e], top);
      }
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[n][d][i] *= f[i & 1];
          if (warp >= 2) part(warp - 2, n, d, i) = acc[n][d][i];
        }
    }
    __syncthreads();
    if (warp < 2) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) part(warp, n, d, i) += acc[n][d][i];
    }
    __syncthreads();
    few_finish<T, D, M, Cfg>(p, w, it, merge, row_stats, [](int, int, float) { return 1.f; });
    __syncthreads();                                     // the results may be replaced
  }
  copy_wait<0>();
}

template <int D, int M>
__global__ void __launch_bounds__(kFewWarps * 32, FewCfg<float, D, M>::kBlocks)
paged_few_f32_kernel(const __grid_constant__ PagedAttnParams p, const WorkPartials w, int least, uint32_t slope, int whole) {
  using T = float;
  using Cfg = FewCfg<T, D, M>;
  constexpr int E = D / 32, C = Cfg::kChunks;
  extern __shared__ __align__(128) uint8_t few_smem[];
  float* merge = reinterpret_cast<float*>(few_smem + Cfg::kOffMerge);          // [warps][M][D]
  float* qs = reinterpret_cast<float*>(few_smem + Cfg::kOffQ);
  float* stat = reinterpret_cast<float*>(few_smem + Cfg::kOffStat);
  uint32_t* masks = reinterpret_cast<uint32_t*>(stat + kFewWarps * M * 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dependency_wait();
  allow_dependents();
  const WorkShare share = find_share<M, Cfg::KT, 1, 8>(p, least, slope, whole);
  publish_share(share, w);
  FewLoader<T, D, M> load;
  load.ring = smem_addr(few_smem) + warp * Cfg::kRing;
  load.masks = masks + warp * Cfg::kStages;
  load.start(p, share, warp, lane);
#pragma unroll 1
  for (int s = 0; s < Cfg::kStages; ++s) load.issue(p, s, warp, lane);
  WorkIter<M, Cfg::KT> iter;
  iter.start(share);
  WorkItem it;
  int stage = 0, tok, head;
  while (iter.next(p, it)) {
    int lim[M];
#pragma unroll
    for (int g = 0; g < M; ++g) {
      row_of<M>(p, it, g, tok, head);
      lim[g] = g < it.rows ? visible_keys(it.x, tok) : INT32_MAX;
    }
    for (int i = threadIdx.x; i < M * D; i += kFewWarps * 32) {
      const int g = i / D;
      row_of<M>(p, it, g, tok, head);
      qs[i] = g < it.rows ? ((const float*)p.q)[(int64_t)(it.x.q0 + tok) * p.sq.s + (int64_t)head * p.sq.h + i % D] * p.scale_log2 : 0.f;
    }
    __syncthreads();
    float acc[M][E], m[M], l[M];
#pragma unroll
    for (int g = 0; g < M; ++g) {
      m[g] = -INFINITY;
      l[g] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] = 0.f;
    }
#pragma unroll 1
    for (int kt = it.k0; kt < it.k1; ++kt) {
      copy_wait<Cfg::kStages - 1>();
      __syncwarp();
      const uint32_t mask = load.masks[stage];
      if (mask) {
        const uint8_t* kb = few_smem + warp * Cfg::kRing + stage * 2 * Cfg::kTile;
        const uint8_t* vb = kb + Cfg::kTile;
        const int row = lane & 7, part = lane >> 3;
        float s[M];
#pragma unroll
        for (int g = 0; g < M; ++g) s[g] = 0.f;
#pragma unroll
        for (int i = 0; i < C / 4; ++i) {
          const int c = part * (C / 4) + i;
          const float4 k = *reinterpret_cast<const float4*>(kb + (row * C + (c ^ row)) * 16);
#pragma unroll
          for (int g = 0; g < M; ++g) {
            const float4 q = *reinterpret_cast<const float4*>(qs + g * D + c * 4);
            s[g] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[g]))));
          }
        }
        const int key = kt * Cfg::KT + warp * Cfg::kRows + row;
        const bool there = (mask >> row) & 1;
#pragma unroll
        for (int g = 0; g < M; ++g) {
          s[g] += __shfl_xor_sync(0xffffffffu, s[g], 8);
          s[g] += __shfl_xor_sync(0xffffffffu, s[g], 16);
          if (!there || key >= lim[g]) s[g] = -INFINITY;
          float x = s[g];
#pragma unroll
          for (int o = 1; o < 8; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
          x = fmaxf(x, m[g]);
          const float c = m[g] == -INFINITY ? 0.f : exp2f(m[g] - x);
          m[g] = x;
          s[g] = exp2f(s[g] - (x == -INFINITY ? 0.f : x));       // the weight
          l[g] = l[g] * c + s[g];                                // of this lane's keys; the four quarters hold the same
#pragma unroll
          for (int e = 0; e < E; ++e) acc[g][e] *= c;
        }
#pragma unroll
        for (int j = 0; j < Cfg::kRows; ++j) {
          float v[E];
          const int at = lane * E / 4, in = lane * E % 4;
          const float* src = reinterpret_cast<const float*>(vb + (j * C + (at ^ j)) * 16) + in;
#pragma unroll
          for (int e = 0; e < E; ++e) v[e] = src[e];
#pragma unroll
          for (int g = 0; g < M; ++g) {
            const float pj = __shfl_sync(0xffffffffu, s[g], j);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[g][e] = fmaf(pj, v[e], acc[g][e]);
          }
        }
      }
      __syncwarp();
      load.issue(p, stage, warp, lane);
      stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;
    }
#pragma unroll
    for (int g = 0; g < M; ++g) {
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], o);
#pragma unroll
      for (int e = 0; e < E; ++e) merge[(warp * M + g) * Cfg::kPitch + lane * E + e] = acc[g][e];
      if (lane == 0) { stat[warp * M + g] = m[g]; stat[(kFewWarps + warp) * M + g] = l[g]; }
    }
    __syncthreads();
    auto factor = [&](int v, int g, float top) { return part_weight(stat[v * M + g], stat[(kFewWarps + v) * M + g], top); };
    auto row_stats = [&](int g, float& top, float& sum) {
      top = -INFINITY;
      sum = 0.f;
#pragma unroll
      for (int v = 0; v < kFewWarps; ++v) top = fmaxf(top, stat[v * M + g]);
#pragma unroll
      for (int v = 0; v < kFewWarps; ++v) sum = fmaf(stat[(kFewWarps + v) * M + g], factor(v, g, top), sum);
    };
    few_finish<T, D, M, Cfg>(p, w, it, merge, row_stats, factor);
    __syncthreads();                                 // queries, sums and results may be replaced
  }
  copy_wait<0>();
}

template <typename T, int D, int M>
static int launch_few(const PagedAttnParams& p, cudaStream_t st) {
  using Cfg = FewCfg<T, D, M>;
  auto kern = [] { if constexpr (Cfg::kHalf) return paged_few_half_kernel<T, D, M>; else return paged_few_f32_kernel<D, M>; }();
  static SmemLimit limit;
  if (int rc = limit.raise((const void*)kern, Cfg::kSmem)) return rc;
  const int grid = Cfg::kBlocks * sm_count();
  // Tables that end within a few tiles: no item is cut then, and there is nothing to join (a second launch costs 3 us, as
  // much as six tiles one after the other). The host knows the table's width and not the lengths: one request of 144 keys, 12 heads of
  // 64 in fp32, takes 16 us with a table cut to its size and 22 with one of 2048 positions.
  const int whole = (int64_t)p.width * p.page.d <= 6 * Cfg::KT;
  TempBuf part(whole ? 0 : partial_bytes(grid, M, D), st, Scratch::kOwnPool);
  if (!part.ok()) return MT_ERR_CUDA;
  const WorkPartials w = whole ? WorkPartials{} : partials_in(part.ptr, grid, M, D);
  MT_CHECK_CUDA(launch_overlapped(kern, dim3((unsigned)grid), dim3(kFewWarps * 32), Cfg::kSmem, st, p, w, 3, tile_slope<M, Cfg::KT>(p.group), whole));
  count_launch();
  return whole ? MT_OK : launch_join<T, D, M, Cfg::KT>(p, w, grid, st);
}

template <typename T, int D>
static int launch_few_rows(const PagedAttnParams& p, int64_t rows, cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (rows <= 8) return launch_few<T, D, 8>(p, st);
    // More rows than 16 read keys and values again (from L2) for each 16: tiles of 24 and 32 rows need 255 registers and take
    // longer where latency counts (20 rows, 16 x 500..2000 keys x 128: 26.6 us against 22.7; 28 rows, 8 x 200..900: 29.3 against
    // 19.2) and gain 7 % where bandwidth does (20 rows, 64 requests: 43.0 against 46.1).
    return launch_few<T, D, 16>(p, st);
  } else {
    // Shares are weighed in 64 bits: tiles^2 / 2 * 2^11 M / group, which passes them between 2^27 and 2^28 rows of a request
    // where M group <= 4.
    if ((int64_t)p.rows * p.group >= 1 << 27) return launch_few<T, D, 8>(p, st);
    if (rows <= 1) return launch_few<T, D, 1>(p, st);
    if (rows <= 2) return launch_few<T, D, 2>(p, st);
    if (rows <= 4) return launch_few<T, D, 4>(p, st);
    return launch_few<T, D, 8>(p, st);
  }
}

int attn_paged_few(const PagedAttnParams& p, int64_t row_hint, int head_dim, int dtype, cudaStream_t st) {
  MT_DISPATCH_FLOAT(dtype, T, return head_dim == 64 ? (launch_few_rows<T, 64>(p, row_hint, st)) : (launch_few_rows<T, 128>(p, row_hint, st)));
  return MT_OK;
}

}  // namespace mt
