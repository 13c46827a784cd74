// Attention over pages in fp32 for many query rows (prompts and chunks; few rows: attention_paged_few.cu).
//
// CUDA cores: 4 D operations per (row, visible key), so the FMA rate is the bound. A block of four warps has
// 64 query rows (tokens times the query heads of the group) and walks key tiles of KT = 4096 / D keys, two stages
// filled by 16-byte cp.async (row addresses through the request's table; zeros for rows that are not there). A
// warp owns 16 rows, a thread 4 rows x KT/8 keys of the scores and 4 rows x D/8 columns of the output,
// both by packed FMAs (two per instruction) on float4 loads: 12 wide loads per 64 packed FMAs for the scores, no
// bank conflicts (16-byte pieces swizzled by row). Row statistics live in the 8 threads that share a row, and the weights cross
// to the output's layout through shared memory of the warp's own, so a tile costs two block barriers.
// Prompts of 100..500 tokens, 12 heads of 64: 48 us (12 TFLOP/s; 60 items of 64 rows per request and little to hide latency behind).
#include "attention_paged.cuh"
#include "paged_work.cuh"
#include "attention_tc.cuh"
#include "tempbuf.cuh"

namespace mt {

constexpr int kPfM = 64, kPfThreads = 128;

template <int D> struct PfCfg {
  static constexpr int KT = 4096 / D;                    // 64 or 32 keys
  static constexpr int C = D / 4;                        // 16-byte pieces of a row
  static constexpr int kTile = KT * D * 4;               // 16 KB
  static constexpr int kPitch = KT + 4;                  // of a row of weights, floats
  static constexpr int kOffRing = kPfM * D * 4;          // behind the queries: two stages of keys and values
  static constexpr int kOffP = kOffRing + 4 * kTile;
  static constexpr int kOffThere = kOffP + kPfM * kPitch * 4;   // [2 stages][KT]: is the row there
  static constexpr int kSmem = kOffThere + 2 * KT;
  static_assert(2 * (kSmem + 1024 + 384) <= 233472, "two blocks per SM");
};

template <int D>
__global__ void __launch_bounds__(kPfThreads, 2)
paged_f32_kernel(const __grid_constant__ PagedAttnParams p, const WorkPartials w, int least, uint32_t slope) {
  using Cfg = PfCfg<D>;
  constexpr int KT = Cfg::KT, C = Cfg::C, NK = KT / 8, NO = D / 32;   // keys, and float4 columns, of a thread
  extern __shared__ __align__(128) uint8_t pf_smem[];
  float* ps = reinterpret_cast<float*>(pf_smem + Cfg::kOffP);
  uint8_t* there = pf_smem + Cfg::kOffThere;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cg = lane & 7, row0 = warp * 16 + (lane >> 3) * 4;        // this thread's first row of the tile
  grid_dependency_wait();
  allow_dependents();
  const WorkShare share = find_share<kPfM, KT, 1, 8>(p, least, slope, false);
  publish_share(share, w);
  WorkIter<kPfM, KT> iter;
  iter.start(share);
  WorkItem it;
  while (iter.next(p, it)) {
    const int32_t* table = p.tables + (int64_t)it.r * p.width;
    auto issue = [&](int kt, int stage) {
      const uint32_t kd = (uint32_t)__cvta_generic_to_shared(pf_smem + Cfg::kOffRing + stage * 2 * Cfg::kTile);
#pragma unroll 4
      for (int i = 0; i < KT * C / kPfThreads; ++i) {
        const int row = (i * kPfThreads + (int)threadIdx.x) / C, c = (int)threadIdx.x % C, key = kt * KT + row;
        const int64_t off = key < it.keys ? paged_row(p, table, key) : -1;
        const int64_t src = off >= 0 ? off + (int64_t)it.hk * p.sc.h + c * 4 : 0;
        const int to = (row * C + (c ^ (row & 7))) * 16;
        copy16_async(kd + to, (const float*)p.kp + src, off >= 0 ? 16 : 0);
        copy16_async(kd + Cfg::kTile + to, (const float*)p.vp + src, off >= 0 ? 16 : 0);
        if (c == 0) there[stage * KT + row] = off >= 0;
      }
      copy_commit();
    };
    if (it.k0 < it.k1) issue(it.k0, 0);
    // queries, scaled, rows swizzled by groups of four; and what this thread's rows see
    for (int i = threadIdx.x; i < kPfM * C; i += kPfThreads) {
      const int row = i / C, c = i % C;
      int token, head;
      row_of<kPfM>(p, it, row, token, head);
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < it.rows) {
        const float* q = (const float*)p.q + (int64_t)(it.x.q0 + token) * p.sq.s + (int64_t)head * p.sq.h + c * 4;
        v = make_float4(q[0] * p.scale_log2, q[1] * p.scale_log2, q[2] * p.scale_log2, q[3] * p.scale_log2);
      }
      *reinterpret_cast<float4*>(pf_smem + (row * C + (c ^ ((row >> 2) & 7))) * 16) = v;
    }
    int lim[4], token, head;
    float m[4], l[4];
    uint64_t o[4][NO][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      row_of<kPfM>(p, it, row0 + i, token, head);
      lim[i] = row0 + i < it.rows ? visible_keys(it.x, token) : INT32_MAX;
      m[i] = -INFINITY;
      l[i] = 0.f;
#pragma unroll
      for (int j = 0; j < NO; ++j) o[i][j][0] = o[i][j][1] = 0ull;
    }
    for (int kt = it.k0; kt < it.k1; ++kt) {
      const int stage = (kt - it.k0) & 1;
      if (kt + 1 < it.k1) {
        issue(kt + 1, stage ^ 1);
        copy_wait<1>();
      } else {
        copy_wait<0>();
      }
      __syncthreads();
      const uint8_t* kb = pf_smem + Cfg::kOffRing + stage * 2 * Cfg::kTile;
      const uint8_t* vb = kb + Cfg::kTile;
      uint64_t s2[4][NK];                                // sums over even and odd elements of head_dim
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < NK; ++j) s2[i][j] = 0ull;
#pragma unroll 2
      for (int c = 0; c < C; ++c) {
        ulonglong2 q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const ulonglong2*>(pf_smem + ((row0 + i) * C + (c ^ ((row0 >> 2) & 7))) * 16);
#pragma unroll
        for (int j = 0; j < NK; ++j) {                   // keys cg, cg + 8, ...
          const ulonglong2 k = *reinterpret_cast<const ulonglong2*>(kb + ((cg + 8 * j) * C + (c ^ cg)) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) s2[i][j] = f2_fma(q[i].y, k.y, f2_fma(q[i].x, k.x, s2[i][j]));
        }
      }
      const int key0 = kt * KT;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float s[NK], x = m[i];
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          float a, b;
          f2_unpack(s2[i][j], a, b);
          s[j] = a + b;
          const int at = cg + 8 * j;
          if (key0 + at >= lim[i] || !there[stage * KT + at]) s[j] = -INFINITY;
          x = fmaxf(x, s[j]);
        }
#pragma unroll
        for (int b = 1; b < 8; b <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, b));
        const float c = m[i] == -INFINITY ? 0.f : exp2f(m[i] - x), u = x == -INFINITY ? 0.f : x;
        m[i] = x;
        l[i] *= c;
        const uint64_t c2 = f2_pack(c, c);
#pragma unroll
        for (int j = 0; j < NO; ++j) { o[i][j][0] = f2_mul(o[i][j][0], c2); o[i][j][1] = f2_mul(o[i][j][1], c2); }
#pragma unroll
        for (int j = 0; j < NK; ++j) {
          const float e = exp2f(s[j] - u);
          l[i] += e;
          ps[(row0 + i) * Cfg::kPitch + cg + 8 * j] = e;
        }
      }
      __syncwarp();
#pragma unroll 2
      for (int k4 = 0; k4 < KT; k4 += 4) {
        float4 e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = *reinterpret_cast<const float4*>(ps + (row0 + i) * Cfg::kPitch + k4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          ulonglong2 v[NO];
#pragma unroll
          for (int j = 0; j < NO; ++j) v[j] = *reinterpret_cast<const ulonglong2*>(vb + ((k4 + k) * C + ((cg + 8 * j) ^ ((k4 + k) & 7))) * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f = k == 0 ? e[i].x : k == 1 ? e[i].y : k == 2 ? e[i].z : e[i].w;
            const uint64_t f2 = f2_pack(f, f);
#pragma unroll
            for (int j = 0; j < NO; ++j) { o[i][j][0] = f2_fma(f2, v[j].x, o[i][j][0]); o[i][j][1] = f2_fma(f2, v[j].y, o[i][j][1]); }
          }
        }
      }
      __syncthreads();                                   // the stage may be filled again
    }
    const int slot = partial_slot(it);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int b = 1; b < 8; b <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], b);
      const int row = row0 + i;
      row_of<kPfM>(p, it, row, token, head);
      const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
      bool nan = false;
#pragma unroll
      for (int j = 0; j < NO; ++j) {
        float4 v;
        f2_unpack(o[i][j][0], v.x, v.y);
        f2_unpack(o[i][j][1], v.z, v.w);
        if (row >= it.rows) continue;
        const int col = (cg + 8 * j) * 4;
        if (slot >= 0) {
          *reinterpret_cast<float4*>(w.o + ((int64_t)slot * kPfM + row) * D + col) = v;
          continue;
        }
        v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
        nan |= isnan(v.x) || isnan(v.y) || isnan(v.z) || isnan(v.w);
        float* to = (float*)p.o + (int64_t)(it.x.q0 + token) * p.so.s + (int64_t)head * p.so.h + col;
        if (p.o_quads) *reinterpret_cast<float4*>(to) = v;
        else { to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w; }
      }
      if (slot >= 0 && cg == 0 && row < it.rows)
        *reinterpret_cast<float2*>(w.ml + ((int64_t)slot * kPfM + row) * 2) = make_float2(m[i], l[i]);
      uint32_t again = __ballot_sync(0xffffffffu, nan);
      while (again) {                                    // rows with NaN, eight lanes each
        const int at = __ffs((int)again) - 1;
        again &= ~(0xffu << (at & ~7));
        const int t = __shfl_sync(0xffffffffu, token, at), h = __shfl_sync(0xffffffffu, head, at);
        __syncwarp();
        paged_row_plain<float, D>(p, it.x, it.r, t, h);
      }
    }
    __syncthreads();                                     // the queries may be replaced
  }
}

template <int D>
static int launch_paged_f32(const PagedAttnParams& p, cudaStream_t st) {
  using Cfg = PfCfg<D>;
  auto kern = paged_f32_kernel<D>;
  static SmemLimit limit;
  if (int rc = limit.raise((const void*)kern, Cfg::kSmem)) return rc;
  const int grid = 2 * sm_count();
  TempBuf part(partial_bytes(grid, kPfM, D), st, Scratch::kOwnPool);
  if (!part.ok()) return MT_ERR_CUDA;
  const WorkPartials w = partials_in(part.ptr, grid, kPfM, D);
  MT_CHECK_CUDA(launch_overlapped(kern, dim3((unsigned)grid), dim3(kPfThreads), Cfg::kSmem, st, p, w, 3, tile_slope<kPfM, Cfg::KT>(p.group)));
  count_launch();
  return launch_join<float, D, kPfM, Cfg::KT>(p, w, grid, st);
}

int attn_paged_f32(const PagedAttnParams& p, int head_dim, cudaStream_t st) {
  return head_dim == 64 ? launch_paged_f32<64>(p, st) : launch_paged_f32<128>(p, st);
}

}  // namespace mt
