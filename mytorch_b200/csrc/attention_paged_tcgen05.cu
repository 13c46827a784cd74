// Attention over pages on the tensor cores, fp16/bf16: prompts, chunks of prompts and batches that mix
// them with decoding requests.
//
// Persistent, one CTA per SM, 416 threads; a CTA walks its share of the work (paged_work.cuh). An item is
// 256 query rows (tokens times the query heads of the group, so grouped heads fill tiles and share the loads) of one
// key/value head, in two subtiles A and B of 128, against key tiles of 128:
//   warps 8-11  loaders: key and value rows lie wherever their pages are, so they come by 16-byte cp.async
//               (a thread looks up one row's page, a tile ahead, and hands the address to the lanes that copy it),
//               written in the 128-byte swizzle that the MMA reads, into one ring in the order of use
//               K0 K1 V0 K2 V1 ...; two groups stay in flight behind the one being queued. Rows behind the
//               last key or on a bad page are zeros, their bits in a mask of the tile are clear.
//   warp 12     MMA issuer: S_A = Q_A K^T and S_B = Q_B K^T into tensor memory, then per tile O_A += P_A V and the
//               next S_A while subtile B is in its softmax, O_B += P_B V and the next S_B while A is: the
//               tensor pipe always has the other subtile's products.
//   warps 0-3, 4-7  softmax of A and B: a thread owns a row (TMEM lane), reads its 128 scores twice (maximum;
//               weights) in pieces of 32, and writes the weights as packed half pairs over the scores, which
//               nobody reads any more; P is the A operand straight from tensor memory. The running maximum
//               only moves, and O in tensor memory is only rescaled, when it grew by more than 2^8. The
//               weights are rounded to the type for the product (half a step, as the output is); sums are fp32.
// Tensor memory: S_A, S_B (128 columns each), O_A, O_B (D each).
//
// Roofline: tensor pipe, 4 D operations per (row, visible key), or the exponentials (16 per clock per SM,
// 1024 cycles per 128x128 tile, the MMA's time at D = 128 and twice it at D = 64).
#include "attention_paged.cuh"
#include "paged_work.cuh"
#include "attention_tc.cuh"
#include "tempbuf.cuh"

namespace mt {

using namespace sm100;

constexpr int kPtM = 256, kPtKT = 128;
constexpr int kPtThreads = 416;
constexpr int kPtAbort = 105;

template <int D> struct PtCfg {
  static constexpr int kChunks = D / 64;                 // 64-column (128-byte) slices of head_dim
  static constexpr int kTile = 128 * D * 2;              // 128 rows of Q, K or V
  static constexpr int kRing = D == 128 ? 5 : 8;
  static constexpr int kOffRing = 2 * kTile;             // behind Q_A and Q_B
  static constexpr int kOffBar = kOffRing + kRing * kTile;
  static constexpr int kOffMask = kOffBar + 256;         // [16 tiles][4 words]
  static constexpr int kSmem = kOffMask + 256;
  static constexpr int kColO = 256;
  static_assert(kSmem + 1024 <= 232448, "shared memory of one CTA, static part included");
};

// Key tiles of the item that subtile s works on, as a count from it.k0.
__device__ __forceinline__ int subtile_tiles(const PagedAttnParams& p, const WorkItem& it, int s) {
  if (it.rows <= 128 * s) return 0;
  const int64_t rows = min((int64_t)it.t * kPtM + 128 * (s + 1), (int64_t)it.x.n_new * p.group);
  const int n = (visible_keys(it.x, (int)p.by_group.div((uint32_t)(rows - 1))) + kPtKT - 1) / kPtKT;
  return max(0, min(n, it.k1) - it.k0);
}

__device__ __forceinline__ void pt_copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int D, typename T>
__global__ void __launch_bounds__(kPtThreads, 1)
paged_tc_kernel(const __grid_constant__ PagedAttnParams p, const WorkPartials w, int least, uint32_t slope, int is_bf16, int q_vec, int o_vec) {
  using Cfg = PtCfg<D>;
  constexpr int kRing = Cfg::kRing;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = smem_u32(smem_raw);
  if (base & 1023u) {   // the 128-byte swizzle needs 1024-byte aligned tiles
    if (threadIdx.x == 0 && p.flag) atomicMax(p.flag, kPtAbort);
    return;
  }
  const uint32_t bar0 = base + Cfg::kOffBar;
  const uint32_t bar_full0 = bar0, bar_empty0 = bar0 + 64, bar_q = bar0 + 128, bar_qfree = bar0 + 136, bar_s0 = bar0 + 144,
                 bar_p0 = bar0 + 160, bar_o0 = bar0 + 176;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + Cfg::kOffBar + 192);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_raw + Cfg::kOffBar + 196);
  volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(smem_raw + Cfg::kOffMask);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) { mbar_init(bar_full0 + 8 * i, 4); mbar_init(bar_empty0 + 8 * i, 1); }
    mbar_init(bar_q, 4);
    mbar_init(bar_qfree, 1);
    for (int s = 0; s < 2; ++s) { mbar_init(bar_s0 + 8 * s, 1); mbar_init(bar_p0 + 8 * s, 4); mbar_init(bar_o0 + 8 * s, 1); }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
  }
  if (warp == 12) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  grid_dependency_wait();
  allow_dependents();
  const WorkShare share = find_share<kPtM, kPtKT>(p, least, slope);
  publish_share(share, w);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  WorkIter<kPtM, kPtKT> iter;
  iter.start(share);
  WorkItem it;

  if (warp >= 8 && warp < 12) {
    // ------------------------------------------------------------- loaders --
    const int lw = warp - 8;
    uint32_t pend0 = 0, pend1 = 0;                       // barriers of the copy groups in flight, oldest first
    auto announce = [&](uint32_t bar) {                  // the copies have landed: make them visible to the MMA
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto push = [&](uint32_t bar) {
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (pend0) {
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        announce(pend0);
      }
      pend0 = pend1;
      pend1 = bar;
    };
    auto drain = [&]() {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      if (pend0) announce(pend0);
      if (pend1) announce(pend1);
      pend0 = pend1 = 0;
    };
    // A wait that would block first hands over what is in flight, which the other side may be waiting for.
    auto wait_for = [&](uint32_t bar, uint32_t parity) -> bool {
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
      drain();
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
    };
    int used = 0, tiles = 0;                             // ring slots and key tiles so far
    auto copy_rows = [&](uint32_t dst, const T* src, int64_t off) {   // this warp's 32 rows, off: this lane's row
      constexpr int C = D / 8;                           // 16-byte pieces of a row
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int r = (i * 32 + lane) / C, c = (i * 32 + lane) % C;
        const int64_t o = __shfl_sync(0xffffffffu, off, r);
        const int row = lw * 32 + r;
        pt_copy16(dst + (c >> 3) * 16384 + row * 128 + (((c & 7) ^ (row & 7)) << 4), src + (o >= 0 ? o + c * 8 : 0), o >= 0 ? 16 : 0);
      }
    };
    auto into_ring = [&](const T* src, int64_t off) -> bool {
      const int slot = used % kRing;
      if (!wait_for(bar_empty0 + 8 * slot, ((used / kRing) & 1) ^ 1u)) return false;
      copy_rows(base + Cfg::kOffRing + slot * Cfg::kTile, src, off);
      push(bar_full0 + 8 * slot);
      ++used;
      return true;
    };
    bool ok = true;
    for (int tn = 0; ok && iter.next(p, it); ++tn) {
      const int n = max(subtile_tiles(p, it, 0), subtile_tiles(p, it, 1));
      if (n == 0) { --tn; continue; }                    // no key: the softmax warps write zeros
      const int32_t* table = p.tables + (int64_t)it.r * p.width;
      const int64_t head = (int64_t)it.hk * p.sc.h;
      auto page_at = [&](int kt) {                       // of this lane's row of the tile; -1: none
        const int key = kt * kPtKT + lw * 32 + lane;
        if (kt >= it.k0 + n || key >= it.keys) return -1;
        const int page = table[p.page.div((uint32_t)key)];
        if ((unsigned)page < (unsigned)p.n_pages) return page;
        if (p.flag) atomicMax(p.flag, kPagedFlag);
        return -1;
      };
      auto row_at = [&](int kt, int page) -> int64_t {
        const uint32_t key = (uint32_t)(kt * kPtKT + lw * 32 + lane);
        return page >= 0 ? (int64_t)page * p.sc.b + (int64_t)(key - p.page.div(key) * p.page.d) * p.sc.s + head : -1;
      };
      auto load_k = [&](int64_t off) -> bool {
        const uint32_t mask = __ballot_sync(0xffffffffu, off >= 0);
        if (lane == 0) masks[(tiles & 15) * 4 + lw] = mask;
        ++tiles;
        return into_ring((const T*)p.kp, off);
      };
      int64_t off = row_at(it.k0, page_at(it.k0)), off_next = -1;
      int page = page_at(it.k0 + 1);
      if (!(ok = load_k(off))) break;
      // queries, once the last score MMA of the item before has read them
      if (tn > 0 && !(ok = wait_for(bar_qfree, (tn - 1) & 1))) break;
#pragma unroll 1
      for (int s = 0; s < 2; ++s) {
        const int row = s * 128 + lw * 32 + lane;
        int token, h;
        row_of<kPtM>(p, it, row, token, h);
        const int64_t q = row < it.rows ? (int64_t)(it.x.q0 + token) * p.sq.s + (int64_t)h * p.sq.h : -1;
        const uint32_t dst = base + s * Cfg::kTile;
        if (q_vec) copy_rows(dst, (const T*)p.q, q);
        else {                                           // rows at any address: element by element
          for (int c = 0; c < D; ++c) {
            const int r = lw * 32 + lane;
            T* to = reinterpret_cast<T*>(smem_raw + s * Cfg::kTile + (c >> 6) * 16384 + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4)) + (c & 7);
            *to = q >= 0 ? ((const T*)p.q)[q + c] : from_f<T>(0.f);
          }
        }
      }
      push(bar_q);
      for (int i = 0; i < n; ++i) {
        if (i + 1 < n) {
          off_next = row_at(it.k0 + i + 1, page);
          page = page_at(it.k0 + i + 2);
          if (!(ok = load_k(off_next))) break;
        }
        if (!(ok = into_ring((const T*)p.vp, off))) break;
        off = off_next;
      }
    }
    drain();
  } else if (warp == 12) {
    // ---------------------------------------------------------- MMA issuer --
    if (lane == 0) {
      const uint32_t idesc_s = idesc_f16(is_bf16, 0, 0, 128, 128);
      const uint32_t idesc_o = idesc_f16(is_bf16, 0, 1, 128, D);
      uint64_t dq[4 * Cfg::kChunks], dk0[4 * Cfg::kChunks], dv0[8];     // of Q_A and of ring slot 0
#pragma unroll
      for (int c = 0; c < Cfg::kChunks; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          dq[c * 4 + k] = smem_desc_sw128(base + c * 16384 + k * 32, 16, 1024);
          dk0[c * 4 + k] = smem_desc_sw128(base + Cfg::kOffRing + c * 16384 + k * 32, 16, 1024);
        }
#pragma unroll
      for (int k = 0; k < 8; ++k) dv0[k] = smem_desc_sw128(base + Cfg::kOffRing + k * 2048, 16384, 1024);
      int used = 0, np[2] = {0, 0};                      // ring slots taken; weight tiles awaited per subtile
      auto wait_full = [&](int u) { return mbar_wait(bar_full0 + 8 * (u % kRing), (u / kRing) & 1, abort_flag); };
      auto issue_s = [&](int s, int slot) {
        uint64_t a[4 * Cfg::kChunks], b[4 * Cfg::kChunks];
#pragma unroll
        for (int k = 0; k < 4 * Cfg::kChunks; ++k) {
          a[k] = dq[k] + (uint64_t)(s * Cfg::kTile >> 4);
          b[k] = dk0[k] + (uint64_t)(slot * Cfg::kTile >> 4);
        }
        umma_f16_x4(tmem_base + 128 * s, a, b, idesc_s, 0u);
        if (Cfg::kChunks == 2) umma_f16_x4(tmem_base + 128 * s, a + 4 * (Cfg::kChunks - 1), b + 4 * (Cfg::kChunks - 1), idesc_s, 1u);
        umma_commit(bar_s0 + 8 * s);
      };
      bool ok = true;
      for (int tn = 0; ok && iter.next(p, it); ++tn) {
        const int count[2] = {subtile_tiles(p, it, 0), subtile_tiles(p, it, 1)};
        const int n = max(count[0], count[1]);
        if (n == 0) { --tn; continue; }
        int uk = used++;                                 // slot of the next key tile
        if (!wait_full(uk) || !mbar_wait(bar_q, tn & 1, abort_flag)) break;
        tc_fence_after();
        for (int s = 0; s < 2; ++s)
          if (count[s] > 0) issue_s(s, uk % kRing);
        umma_commit(bar_empty0 + 8 * (uk % kRing));
        if (n == 1) umma_commit(bar_qfree);
        for (int i = 0; i < n; ++i) {
          const bool more = i + 1 < n;
          if (more) uk = used++;
          const int uv = used++;
          uint64_t b[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) b[k] = dv0[k] + (uint64_t)((uv % kRing) * Cfg::kTile >> 4);
          if (more && !wait_full(uk)) { ok = false; break; }
          if (!wait_full(uv)) { ok = false; break; }
          for (int s = 0; s < 2; ++s) {
            if (i >= count[s]) continue;
            if (!mbar_wait(bar_p0 + 8 * s, np[s] & 1, abort_flag)) { ok = false; break; }
            ++np[s];
            tc_fence_after();
            umma_f16_ts_x8(tmem_base + Cfg::kColO + D * s, tmem_base + 128 * s, b, idesc_o, i > 0 ? 1u : 0u);
            if (i + 1 < count[s]) issue_s(s, uk % kRing);
            else umma_commit(bar_o0 + 8 * s);            // the subtile's last product
          }
          if (!ok) break;
          umma_commit(bar_empty0 + 8 * (uv % kRing));
          if (more) {
            umma_commit(bar_empty0 + 8 * (uk % kRing));
            if (i + 2 == n) umma_commit(bar_qfree);      // the item's last score MMA
          }
        }
      }
      // the last commit signals shared memory: not after the CTA is gone
      if (used > 0) mbar_wait(bar_empty0 + 8 * ((used - 1) % kRing), ((used - 1) / kRing) & 1, abort_flag);
    }
  } else {
    // ------------------------------------------------------------- softmax --
    const int sub = warp >> 2, qtr = warp & 3;
    const int row = sub * 128 + qtr * 32 + lane;         // of the item
    const uint32_t lanes = (uint32_t)(qtr * 32) << 16;
    const uint32_t tmem_s = tmem_base + 128 * sub + lanes, tmem_o = tmem_base + Cfg::kColO + D * sub + lanes;
    int ns = 0, no = 0, tiles = 0;                       // score tiles and items of this subtile so far; key tiles so far
    bool ok = true;
    while (ok && iter.next(p, it)) {
      const int count = subtile_tiles(p, it, sub), n = max(count, subtile_tiles(p, it, sub ^ 1));
      int token, h;
      row_of<kPtM>(p, it, row, token, h);
      const bool real = row < it.rows, busy = it.rows > sub * 128 + qtr * 32;
      const int lim = real ? visible_keys(it.x, token) : INT32_MAX;
      const int lim_min = __reduce_min_sync(0xffffffffu, lim);
      float m = -INFINITY, l = 0.f;
      for (int i = 0; i < count; ++i) {
        const int key0 = (it.k0 + i) * kPtKT;
        if (!__all_sync(0xffffffffu, mbar_wait(bar_s0 + 8 * sub, ns & 1, abort_flag))) { ok = false; break; }
        ++ns;
        tc_fence_after();
        if (!busy) {                                     // no row in this warp: whatever stands in P reaches no other row
          if (lane == 0) mbar_arrive(bar_p0 + 8 * sub);
          continue;
        }
        uint32_t there[4], all = 0xffffffffu;
#pragma unroll
        for (int c = 0; c < 4; ++c) { there[c] = masks[((tiles + i) & 15) * 4 + c]; all &= there[c]; }
        const bool full = all == 0xffffffffu && key0 + kPtKT <= lim_min;
        if (!full) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int left = lim - key0 - 32 * c;        // columns of this piece that the row sees
            if (left < 32) there[c] &= left <= 0 ? 0u : (1u << left) - 1;
          }
        }
        uint32_t r[32];
        float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (!full && !__any_sync(0xffffffffu, there[c] != 0)) continue;
          tmem_ld32(tmem_s + 32 * c, r);
          tmem_ld_wait();
          if (!full) {
#pragma unroll
            for (int e = 0; e < 32; ++e) if (!((there[c] >> e) & 1)) r[e] = 0xff800000u;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            x0 = max3(x0, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
            x1 = max3(x1, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
            x2 = max3(x2, __uint_as_float(r[e + 4]), __uint_as_float(r[e + 5]));
            x3 = max3(x3, __uint_as_float(r[e + 6]), __uint_as_float(r[e + 7]));
          }
        }
        const float top = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * p.scale_log2;
        const bool move = top > m && (m == -INFINITY || top - m > 8.f);
        if (__any_sync(0xffffffffu, move)) {
          const float c = !move ? 1.f : m == -INFINITY ? 0.f : ex2_approx(m - top);
          if (move) { m = top; l *= c; }
          if (i > 0) {                                   // these scores were issued behind the last product into O
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
              tmem_ld32(tmem_o + d, r);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * c);
              tmem_st32(tmem_o + d, r);
            }
          }
        }
        const float sub_m = m == -INFINITY ? 0.f : m;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
          if (full || __any_sync(0xffffffffu, there[c] != 0)) {
            tmem_ld32(tmem_s + 32 * c, r);
            tmem_ld_wait();
            if (!full) {
#pragma unroll
              for (int e = 0; e < 32; ++e) if (!((there[c] >> e) & 1)) r[e] = 0xff800000u;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = ex2_approx(fmaf(__uint_as_float(r[2 * e]), p.scale_log2, -sub_m));
              const float p1 = ex2_approx(fmaf(__uint_as_float(r[2 * e + 1]), p.scale_log2, -sub_m));
              l0 += p0;
              l1 += p1;
              pk[e] = pack2<T>(p0, p1);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) pk[e] = 0u;
          }
          tmem_st16(tmem_s + 16 * c, pk);                // over scores that this thread has read
        }
        l += l0 + l1;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p0 + 8 * sub);
      }
      if (!ok) break;
      tiles += n;
      if (count > 0) {
        if (!__all_sync(0xffffffffu, mbar_wait(bar_o0 + 8 * sub, no & 1, abort_flag))) { ok = false; break; }
        ++no;
        tc_fence_after();
      }
      const int slot = partial_slot(it);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      bool nan = false;
      T* op = (T*)p.o + (real ? (int64_t)(it.x.q0 + token) * p.so.s + (int64_t)h * p.so.h : 0);
      float* po = w.o + ((int64_t)max(slot, 0) * kPtM + row) * D;
      if (busy) {
#pragma unroll 1
        for (int d = 0; d < D; d += 32) {
          uint32_t r[32];
          if (count > 0) {
            tmem_ld32(tmem_o + d, r);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0u;
          }
          if (!real) continue;
          if (slot >= 0) {
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              *reinterpret_cast<float4*>(po + d + e) = make_float4(__uint_as_float(r[e]), __uint_as_float(r[e + 1]),
                                                                   __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
            continue;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) { v[u] = __uint_as_float(r[e + u]) * inv; nan |= isnan(v[u]); }
            if (o_vec)
              *reinterpret_cast<uint4*>(op + d + e) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
            else
              for (int u = 0; u < 8; ++u) op[d + e + u] = from_f<T>(v[u]);
          }
        }
        if (slot >= 0 && real)
          *reinterpret_cast<float2*>(w.ml + ((int64_t)slot * kPtM + row) * 2) = make_float2(m, l);
        uint32_t again = __ballot_sync(0xffffffffu, nan);
        while (again) {
          const int at = __ffs((int)again) - 1;
          again &= again - 1;
          paged_row_plain<T, D>(p, it.x, it.r, __shfl_sync(0xffffffffu, token, at), __shfl_sync(0xffffffffu, h, at));
        }
      }
      tc_fence_before();                                 // O is read: the next item's weights may follow
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag && p.flag) atomicMax(p.flag, kPtAbort);
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D, typename T>
static int launch_paged_tc(const PagedAttnParams& p, cudaStream_t st) {
  using Cfg = PtCfg<D>;
  auto kern = paged_tc_kernel<D, T>;
  static SmemLimit limit;
  if (int rc = limit.raise((const void*)kern, Cfg::kSmem)) return rc;
  const int grid = sm_count();
  TempBuf part(partial_bytes(grid, kPtM, D), st);
  if (!part.ok()) return MT_ERR_CUDA;
  const WorkPartials w = partials_in(part.ptr, grid, kPtM, D);
  auto vec = [](const void* x, mt_strides3 s) { return aligned16(x) && s.h % 8 == 0 && s.s % 8 == 0; };
  MT_CHECK_CUDA(launch_overlapped(kern, dim3((unsigned)grid), dim3(kPtThreads), Cfg::kSmem, st, p, w, 3, tile_slope<kPtM, kPtKT>(p.group),
                                  std::is_same<T, __nv_bfloat16>::value, vec(p.q, p.sq), vec(p.o, p.so)));
  count_launch();
  return launch_join<T, D, kPtM, kPtKT>(p, w, grid, st);
}

int attn_paged_tc(const PagedAttnParams& p, int head_dim, int dtype, cudaStream_t st) {
  if (dtype == MT_F16) return head_dim == 64 ? launch_paged_tc<64, __half>(p, st) : launch_paged_tc<128, __half>(p, st);
  return head_dim == 64 ? launch_paged_tc<64, __nv_bfloat16>(p, st) : launch_paged_tc<128, __nv_bfloat16>(p, st);
}

}  // namespace mt
