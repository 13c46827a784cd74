// Attention over pages for few query rows per key/value head: decoding steps and a few drafted tokens.
//
// HBM bound: every key and value row of a head is read once (2 D bytes a key in half precision, against
// 4 D operations per query row). A block of four warps works on one item at a time: up to 16 rows (tokens times the query
// heads of the group) and a run of key tiles. A warp owns 16 keys (8 in fp32) of each tile and has a ring
// of stages of its own, filled by 16-byte cp.async: page lookups run one tile ahead of the loads,
// loads up to three tiles ahead of the products and on across item boundaries, and no warp waits for
// another until an item's end. Rows that are not there (behind the last key, on a bad page) are
// filled with zeros and masked, so whatever lies in unused rows of a page is never read.
//   half: S = Q K^T and O += P V by mma.sync (m16n8k16). The tensor pipe is idle otherwise (2 % busy), so 1 to 16 rows cost
//         the same, and P goes in as a pair of halves (rounded value and remainder): the weights keep about
//         fp32's precision and the output is as exact as one rounding allows.
//   fp32: lane = key and quarter of head_dim for the scores, lane = elements of head_dim for the output.
// The online softmax is kept per warp; warps join at an item's end through shared memory, blocks through
// the partial results of paged_work.cuh.
#include "attention_paged.cuh"
#include "paged_work.cuh"
#include "tempbuf.cuh"
#include <type_traits>

namespace mt {

constexpr int kFewWarps = 4;

template <typename T, int D, int M> struct FewCfg {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kRows = kHalf ? 16 : 8;                   // keys of a warp in a tile
  static constexpr int KT = kRows * kFewWarps;
  static constexpr int kChunks = D * (int)sizeof(T) / 16;        // 16-byte pieces of a row
  static constexpr int kTile = kRows * kChunks * 16;             // bytes of a warp's keys (or values) of one tile
  static constexpr int kStages = !kHalf && M == 8 && D == 128 ? 2 : 3;
  static constexpr int kRing = kStages * 2 * kTile;              // per warp
  static constexpr int kOffMerge = kFewWarps * kRing;
  static constexpr int kMerge = (kHalf ? 2 : kFewWarps) * M * D * 4;
  static constexpr int kOffQ = kOffMerge + kMerge;               // fp32: the scaled queries
  static constexpr int kOffStat = kOffQ + (kHalf ? 0 : M * D * 4);
  static constexpr int kSmem = kOffStat + kFewWarps * M * 2 * 4 + kFewWarps * kStages * 4;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes global -> shared; with bytes = 0 the destination is zeroed and nothing is read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
template <typename T> __device__ __forceinline__ uint32_t pair_bits(T a, T b) {
  return (uint32_t)*reinterpret_cast<uint16_t*>(&a) | (uint32_t)*reinterpret_cast<uint16_t*>(&b) << 16;
}

// A warp's ring of key and value tiles: the load side of the pipeline.
template <typename T, int D, int M>
struct FewLoader {
  using Cfg = FewCfg<T, D, M>;
  WorkIter<M, Cfg::KT> iter;
  WorkItem it;
  bool valid;
  int kt, page;
  uint32_t ring;
  uint32_t* masks;                       // [stages]: which of the tile's rows are there

  __device__ __forceinline__ void advance(const PagedAttnParams& p, int warp, int lane) {
    while (valid && kt >= it.k1) {
      valid = iter.next(p, it);
      if (valid) kt = it.k0;
    }
    page = -1;
    if (valid) {
      const int key = kt * Cfg::KT + warp * Cfg::kRows + (lane % Cfg::kRows);
      if (key < it.keys) {
        page = p.tables[(int64_t)it.r * p.width + p.page.div((uint32_t)key)];
        if ((unsigned)page >= (unsigned)p.n_pages) {
          if (p.flag) atomicMax(p.flag, kPagedFlag);
          page = -1;
        }
      }
    }
  }
  __device__ __forceinline__ void start(const PagedAttnParams& p, const WorkShare& s, int warp, int lane) {
    iter.start(s);
    it.k1 = 0;
    kt = 0;
    valid = true;
    advance(p, warp, lane);
  }
  // Queues the loads of the tile under the cursor into `stage`, one commit group per call.
  __device__ __forceinline__ void issue(const PagedAttnParams& p, int stage, int warp, int lane) {
    if (valid) {
      const int key = kt * Cfg::KT + warp * Cfg::kRows + (lane % Cfg::kRows);
      const uint32_t in_page = (uint32_t)key - p.page.div((uint32_t)key) * p.page.d;
      const int64_t off = page >= 0 ? (int64_t)page * p.sc.b + (int64_t)in_page * p.sc.s + (int64_t)it.hk * p.sc.h : -1;
      const uint32_t mask = __ballot_sync(0xffffffffu, off >= 0) & ((1u << Cfg::kRows) - 1);
      if (lane == 0) masks[stage] = mask;
      if (mask) {
        const uint32_t kd = ring + stage * 2 * Cfg::kTile, vd = kd + Cfg::kTile;
#pragma unroll
        for (int i = 0; i < Cfg::kRows * Cfg::kChunks / 32; ++i) {
          const int row = (i * 32 + lane) / Cfg::kChunks, c = (i * 32 + lane) % Cfg::kChunks;
          const int64_t o = __shfl_sync(0xffffffffu, off, row);
          const uint32_t to = (row * Cfg::kChunks + (c ^ (row & 7))) * 16;
          const int64_t src = o >= 0 ? o + c * (16 / (int)sizeof(T)) : 0;
          copy16(kd + to, (const T*)p.kp + src, o >= 0 ? 16 : 0);
          copy16(vd + to, (const T*)p.vp + src, o >= 0 ? 16 : 0);
        }
      }
      ++kt;
      advance(p, warp, lane);
    }
    copy_commit();
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kFewWarps * 32, 2)
paged_few_half_kernel(const PagedAttnParams p, const WorkPartials w, int64_t min_weight) {
  constexpr int M = 16;
  using Cfg = FewCfg<T, D, M>;
  extern __shared__ __align__(128) uint8_t few_smem[];
  float* merge = reinterpret_cast<float*>(few_smem + Cfg::kOffMerge);
  float* stat = reinterpret_cast<float*>(few_smem + Cfg::kOffStat);            // [warps][16] maxima, then sums
  uint32_t* masks = reinterpret_cast<uint32_t*>(stat + kFewWarps * M * 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  allow_dependents();
  const WorkShare share = find_share<M, Cfg::KT>(p, min_weight);
  publish_share(share, w);
  FewLoader<T, D, M> load;
  load.ring = smem_addr(few_smem) + warp * Cfg::kRing;
  load.masks = masks + warp * Cfg::kStages;
  load.start(p, share, warp, lane);
#pragma unroll
  for (int s = 0; s < Cfg::kStages; ++s) load.issue(p, s, warp, lane);
  WorkIter<M, Cfg::KT> iter;
  iter.start(share);
  WorkItem it;
  int stage = 0;
  while (iter.next(p, it)) {
    const int ra = lane >> 2, rb = ra + 8;           // this thread's two rows
    int lim_a = INT32_MAX, lim_b = INT32_MAX, tok, head;
    uint32_t qf[D / 16][4];
    row_of<M>(p, it, ra, tok, head);
    const T* qa = (const T*)p.q + (int64_t)(it.x.q0 + tok) * p.sq.s + (int64_t)head * p.sq.h + 2 * (lane & 3);
    if (ra < it.rows) lim_a = visible_keys(it.x, tok);
    row_of<M>(p, it, rb, tok, head);
    const T* qb = (const T*)p.q + (int64_t)(it.x.q0 + tok) * p.sq.s + (int64_t)head * p.sq.h + 2 * (lane & 3);
    if (rb < it.rows) lim_b = visible_keys(it.x, tok);
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      qf[k][0] = ra < it.rows ? pair_bits(qa[k * 16], qa[k * 16 + 1]) : 0u;
      qf[k][1] = rb < it.rows ? pair_bits(qb[k * 16], qb[k * 16 + 1]) : 0u;
      qf[k][2] = ra < it.rows ? pair_bits(qa[k * 16 + 8], qa[k * 16 + 9]) : 0u;
      qf[k][3] = rb < it.rows ? pair_bits(qb[k * 16 + 8], qb[k * 16 + 9]) : 0u;
    }
    float acc[D / 8][4], ma = -INFINITY, mb = -INFINITY, la = 0.f, lb = 0.f;
#pragma unroll
    for (int i = 0; i < D / 8; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    const int first_lim = __shfl_sync(0xffffffffu, lim_a, 0);                  // the tile's first row sees the fewest keys
    for (int kt = it.k0; kt < it.k1; ++kt) {
      copy_wait<Cfg::kStages - 1>();
      __syncwarp();
      const uint32_t mask = load.masks[stage];
      const int key0 = kt * Cfg::KT + warp * Cfg::kRows;
      if (mask) {
        const uint32_t kb = load.ring + stage * 2 * Cfg::kTile, vb = kb + Cfg::kTile;
        float s[2][4] = {};
        {
          const int row = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            uint32_t b[4];
            ldm4(b, kb + (row * Cfg::kChunks + ((2 * k + half) ^ (row & 7))) * 16);
            mma16<T>(s[0], qf[k], b[0], b[1]);
            mma16<T>(s[1], qf[k], b[2], b[3]);
          }
        }
        const bool full = mask == 0xffffu && key0 + 16 <= first_lim;
        float xa = ma, xb = mb;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int j = n * 8 + 2 * (lane & 3) + e;
            s[n][e] *= p.scale_log2;
            s[n][2 + e] *= p.scale_log2;
            if (!full) {
              const bool there = (mask >> j) & 1;
              if (!there || key0 + j >= lim_a) s[n][e] = -INFINITY;
              if (!there || key0 + j >= lim_b) s[n][2 + e] = -INFINITY;
            }
            xa = fmaxf(xa, s[n][e]);
            xb = fmaxf(xb, s[n][2 + e]);
          }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, o));
          xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, o));
        }
        if (__any_sync(0xffffffffu, xa > ma || xb > mb)) {
          const float ca = ma == -INFINITY ? 0.f : exp2f(ma - xa), cb = mb == -INFINITY ? 0.f : exp2f(mb - xb);
          ma = xa;
          mb = xb;
          la *= ca;
          lb *= cb;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) { acc[i][0] *= ca; acc[i][1] *= ca; acc[i][2] *= cb; acc[i][3] *= cb; }
        }
        const float ua = ma == -INFINITY ? 0.f : ma, ub = mb == -INFINITY ? 0.f : mb;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int b = 0; b < 2; ++b) {              // row a, row b
            const float p0 = exp2f(s[n][2 * b] - (b ? ub : ua)), p1 = exp2f(s[n][2 * b + 1] - (b ? ub : ua));
            (b ? lb : la) += p0 + p1;
            const T h0 = from_f<T>(p0), h1 = from_f<T>(p1);
            hi[2 * n + b] = pair_bits(h0, h1);
            lo[2 * n + b] = pair_bits(from_f<T>(p0 - to_f(h0)), from_f<T>(p1 - to_f(h1)));
          }
        const int row = (lane & 7) + (((lane >> 3) & 1) << 3), next = lane >> 4;
#pragma unroll
        for (int c = 0; c < D / 8; c += 2) {
          uint32_t b[4];
          ldm4t(b, vb + (row * Cfg::kChunks + ((c + next) ^ (row & 7))) * 16);
          mma16<T>(acc[c], hi, b[0], b[1]);
          mma16<T>(acc[c + 1], hi, b[2], b[3]);
          mma16<T>(acc[c], lo, b[0], b[1]);
          mma16<T>(acc[c + 1], lo, b[2], b[3]);
        }
      }
      __syncwarp();
      load.issue(p, stage, warp, lane);
      stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;
    }
    // the warps' results: a common maximum, then sums of pairs of warps
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
      la += __shfl_xor_sync(0xffffffffu, la, o);
      lb += __shfl_xor_sync(0xffffffffu, lb, o);
    }
    if ((lane & 3) == 0) {
      stat[warp * M + ra] = ma;
      stat[warp * M + rb] = mb;
      stat[(kFewWarps + warp) * M + ra] = la;
      stat[(kFewWarps + warp) * M + rb] = lb;
    }
    __syncthreads();
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kFewWarps; ++v) {
      top[0] = fmaxf(top[0], stat[v * M + ra]);
      top[1] = fmaxf(top[1], stat[v * M + rb]);
    }
    // without a maximum there are no weights, or only NaN ones, which stay
    auto factor = [](float m, float t, float l) { return m == -INFINITY ? (isnan(l) ? l : 0.f) : exp2f(m - t); };
#pragma unroll
    for (int v = 0; v < kFewWarps; ++v) {
      const float l0 = stat[(kFewWarps + v) * M + ra], l1 = stat[(kFewWarps + v) * M + rb];
      sum[0] = fmaf(l0, factor(stat[v * M + ra], top[0], l0), sum[0]);
      sum[1] = fmaf(l1, factor(stat[v * M + rb], top[1], l1), sum[1]);
    }
    const float fa = factor(ma, top[0], la), fb = factor(mb, top[1], lb);
#pragma unroll
    for (int i = 0; i < D / 8; ++i) { acc[i][0] *= fa; acc[i][1] *= fa; acc[i][2] *= fb; acc[i][3] *= fb; }
    auto hand_over = [&](float* to) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) *reinterpret_cast<float4*>(to + (i * 32 + lane) * 4) = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
    };
    auto take_in = [&](const float* from) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(from + (i * 32 + lane) * 4);
        acc[i][0] += v.x; acc[i][1] += v.y; acc[i][2] += v.z; acc[i][3] += v.w;
      }
    };
    if (warp >= 2) hand_over(merge + (warp - 2) * M * D);
    __syncthreads();
    if (warp < 2) take_in(merge + warp * M * D);
    __syncthreads();
    if (warp == 1) hand_over(merge);
    __syncthreads();
    if (warp == 0) {
      take_in(merge);
      const int slot = partial_slot(it);
      if (slot >= 0) {
        float* po = w.o + (int64_t)slot * M * D;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          *reinterpret_cast<float2*>(po + ra * D + i * 8 + 2 * (lane & 3)) = make_float2(acc[i][0], acc[i][1]);
          *reinterpret_cast<float2*>(po + rb * D + i * 8 + 2 * (lane & 3)) = make_float2(acc[i][2], acc[i][3]);
        }
        if ((lane & 3) == 0) {
          float* ml = w.ml + (int64_t)slot * M * 2;
          *reinterpret_cast<float2*>(ml + 2 * ra) = make_float2(top[0], sum[0]);
          *reinterpret_cast<float2*>(ml + 2 * rb) = make_float2(top[1], sum[1]);
        }
      } else {
        const float ia = sum[0] == 0.f ? 0.f : 1.f / sum[0], ib = sum[1] == 0.f ? 0.f : 1.f / sum[1];
        bool nan_a = false, nan_b = false;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          acc[i][0] *= ia; acc[i][1] *= ia; acc[i][2] *= ib; acc[i][3] *= ib;
          nan_a |= isnan(acc[i][0]) || isnan(acc[i][1]);
          nan_b |= isnan(acc[i][2]) || isnan(acc[i][3]);
        }
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int row = b ? rb : ra;
          row_of<M>(p, it, row, tok, head);
          if (row < it.rows) {
            T* op = (T*)p.o + (int64_t)(it.x.q0 + tok) * p.so.s + (int64_t)head * p.so.h + 2 * (lane & 3);
#pragma unroll
            for (int i = 0; i < D / 8; ++i) { op[i * 8] = from_f<T>(acc[i][2 * b]); op[i * 8 + 1] = from_f<T>(acc[i][2 * b + 1]); }
          }
          uint32_t again = __ballot_sync(0xffffffffu, b ? nan_b : nan_a);
          while (again) {                            // rows with NaN, four lanes each
            const int q = (__ffs((int)again) - 1) >> 2;
            again &= ~(0xfu << (4 * q));
            if (q + 8 * b >= it.rows) continue;
            row_of<M>(p, it, q + 8 * b, tok, head);
            __syncwarp();
            paged_row_plain<T, D>(p, it.x, it.r, tok, head);
          }
        }
      }
    }
  }
  copy_wait<0>();
}

template <int D, int M>
__global__ void __launch_bounds__(kFewWarps * 32, 2)
paged_few_f32_kernel(const PagedAttnParams p, const WorkPartials w, int64_t min_weight) {
  using T = float;
  using Cfg = FewCfg<T, D, M>;
  constexpr int E = D / 32, C = Cfg::kChunks;
  extern __shared__ __align__(128) uint8_t few_smem[];
  float* merge = reinterpret_cast<float*>(few_smem + Cfg::kOffMerge);          // [warps][M][D]
  float* qs = reinterpret_cast<float*>(few_smem + Cfg::kOffQ);
  float* stat = reinterpret_cast<float*>(few_smem + Cfg::kOffStat);
  uint32_t* masks = reinterpret_cast<uint32_t*>(stat + kFewWarps * M * 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  allow_dependents();
  const WorkShare share = find_share<M, Cfg::KT>(p, min_weight);
  publish_share(share, w);
  FewLoader<T, D, M> load;
  load.ring = smem_addr(few_smem) + warp * Cfg::kRing;
  load.masks = masks + warp * Cfg::kStages;
  load.start(p, share, warp, lane);
#pragma unroll
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
      for (int e = 0; e < E; ++e) merge[(warp * M + g) * D + lane * E + e] = acc[g][e];
      if (lane == 0) { stat[warp * M + g] = m[g]; stat[(kFewWarps + warp) * M + g] = l[g]; }
    }
    __syncthreads();
    const int slot = partial_slot(it);
    for (int g = warp; g < it.rows; g += kFewWarps) {
      float top = -INFINITY, sum = 0.f, o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll
      for (int v = 0; v < kFewWarps; ++v) top = fmaxf(top, stat[v * M + g]);
#pragma unroll
      for (int v = 0; v < kFewWarps; ++v) {
        const float mv = stat[v * M + g], lv = stat[(kFewWarps + v) * M + g];
        const float f = mv == -INFINITY ? (isnan(lv) ? lv : 0.f) : exp2f(mv - top);
        sum = fmaf(lv, f, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(merge[(v * M + g) * D + lane * E + e], f, o[e]);
      }
      if (slot >= 0) {
        float* po = w.o + ((int64_t)slot * M + g) * D + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) po[e] = o[e];
        if (lane == 0) *reinterpret_cast<float2*>(w.ml + ((int64_t)slot * M + g) * 2) = make_float2(top, sum);
        continue;
      }
      row_of<M>(p, it, g, tok, head);
      bool nan = false;
#pragma unroll
      for (int e = 0; e < E; ++e) { o[e] = sum == 0.f ? 0.f : o[e] / sum; nan |= isnan(o[e]); }
      if (__any_sync(0xffffffffu, nan)) {
        paged_row_plain<T, D>(p, it.x, it.r, tok, head);
        continue;
      }
      float* op = (float*)p.o + (int64_t)(it.x.q0 + tok) * p.so.s + (int64_t)head * p.so.h + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) op[e] = o[e];
    }
    __syncthreads();                                 // queries, sums and results may be replaced
  }
  copy_wait<0>();
}

template <typename T, int D, int M>
static int launch_few(const PagedAttnParams& p, cudaStream_t st) {
  using Cfg = FewCfg<T, D, M>;
  static_assert(2 * (Cfg::kSmem + 1024 + 320) <= 233472, "two blocks per SM (1 KB each is reserved; 320 bytes of static shared memory)");
  auto kern = [] { if constexpr (Cfg::kHalf) return paged_few_half_kernel<T, D>; else return paged_few_f32_kernel<D, M>; }();
  MT_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
  const int grid = 2 * sm_count();
  TempBuf part(partial_bytes(grid, M, D), st);
  if (!part.ok()) return MT_ERR_CUDA;
  const WorkPartials w = partials_in(part.ptr, grid, M, D);
  kern<<<(unsigned)grid, kFewWarps * 32, Cfg::kSmem, st>>>(p, w, (int64_t)2 * Cfg::KT + kItemKeys);
  MT_LAUNCH_CHECK();
  return launch_join<T, D, M, Cfg::KT>(p, w, grid, st);
}

template <int D>
static int launch_few_f32(const PagedAttnParams& p, int64_t rows, cudaStream_t st) {
  if (rows <= 1) return launch_few<float, D, 1>(p, st);
  if (rows <= 2) return launch_few<float, D, 2>(p, st);
  if (rows <= 4) return launch_few<float, D, 4>(p, st);
  return launch_few<float, D, 8>(p, st);
}

int attn_paged_few(const PagedAttnParams& p, int64_t row_hint, int head_dim, int dtype, cudaStream_t st) {
  if (dtype == MT_F32) return head_dim == 64 ? launch_few_f32<64>(p, row_hint, st) : launch_few_f32<128>(p, row_hint, st);
  if (dtype == MT_F16) return head_dim == 64 ? launch_few<__half, 64, 16>(p, st) : launch_few<__half, 128, 16>(p, st);
  return head_dim == 64 ? launch_few<__nv_bfloat16, 64, 16>(p, st) : launch_few<__nv_bfloat16, 128, 16>(p, st);
}

}  // namespace mt
