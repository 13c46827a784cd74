// Attention over pages on the tensor cores, fp16/bf16: prompts, chunks of prompts and batches that mix
// them with decoding requests.
//
// Persistent, one CTA per SM, 512 threads; a CTA walks its share of the work (paged_work.cuh). An item is
// 256 query rows (tokens times the query heads of the group, so grouped heads fill tiles and share the loads) of one
// key/value head, in two subtiles A and B of 128, against key tiles of 128:
//   warps 8-11  loaders: key and value rows lie wherever their pages are. They come by TMA in boxes that fill pages, 8 rows or
//               more (page sizes that are multiples of 8; zeros for a page outside the pool), each warp a quarter of a tile's
//               boxes: one warp alone takes 5000 cycles to queue the 32 copies of a step with pages of 16 rows, more than the step runs.
//               Other page sizes come by 16-byte cp.async, row by row, in the 128-byte swizzle that the MMA reads. Queries
//               are a box where the heads of a group divide 128, else rows as well. One ring in the order of use,
//               K0 K1 V0 K2 V1 ...; page lookups run a tile ahead; which of a tile's rows are there is a mask next to it.
//   warps 13-15 clear the values behind the last key, where a page's rows may hold anything, before the MMA sees
//               them (such keys are masked as scores).
//   warp 12     MMA issuer: S_A = Q_A K^T and S_B = Q_B K^T into tensor memory, then per tile O_A += P_A V and the
//               next S_A while subtile B is in its softmax, O_B += P_B V and the next S_B while A is: the
//               tensor pipe always has the other subtile's products.
//   warps 0-3, 4-7  softmax of A and B: a thread owns a row (TMEM lane) and holds its 128 scores in registers (the loaders
//               and the issuer hand registers over by setmaxnreg; in pieces of 32 scores, read twice, a tile took 4000 cycles),
//               and writes the weights as packed half pairs over the scores; P is the A operand straight from
//               tensor memory. The running maximum only moves, and O in tensor memory is only rescaled, when it
//               grew by more than 2^8. The weights are rounded to the type for the product (half a step, as
//               the output is); sums are fp32.
// Tensor memory: S_A, S_B (128 columns each), O_A, O_B (D each).
//
// Roofline: tensor pipe, 4 D operations per (row, visible key), or the exponentials (16 per clock per SM,
// 1024 cycles per 128x128 tile, the MMA's time at D = 128 and twice it at D = 64). 2 x 1024 new tokens over 8000..14000 keys, 10/2
// heads of 128, bf16: 138 us, 840 TFLOP/s (a step of 128 keys takes 3400 cycles: a subtile's softmax, 2100, and its products behind
// it, 1340; ordering the subtiles' exponentials changes nothing, a quarter of them as polynomials costs 20 % in instructions).
#include "attention_paged.cuh"
#include "paged_work.cuh"
#include "attention_tc.cuh"
#include "tempbuf.cuh"

namespace mt {

using namespace sm100;

constexpr int kPtM = 256, kPtKT = 128;
constexpr int kPtThreads = 512;
// Registers per thread: 128 at launch; 2 x 128 threads of softmax take what the other 2 x 128 give back.
constexpr int kPtRegsMore = 184, kPtRegsLess = 72;
static_assert(kPtRegsMore + kPtRegsLess <= 2 * 128, "more registers than the block was launched with");
constexpr int kPtAbort = 105;
constexpr int kPtFixed = 4, kPtNear = 16;

template <int D> struct PtCfg {
  static constexpr int kChunks = D / 64;                 // 64-column (128-byte) slices of head_dim
  static constexpr int kTile = 128 * D * 2;              // 128 rows of Q, K or V
  static constexpr int kRing = D == 128 ? 4 : 8;
  static constexpr int kOffRing = 2 * kTile;             // behind Q_A and Q_B
  static constexpr int kOffBar = kOffRing + kRing * kTile;
  static constexpr int kOffMask = kOffBar + 512;         // [16 tiles][4 words]: a bit per row, or per box as the loaders share them
  static constexpr int kOffStage = kOffMask + 512;       // a softmax warp's 32 rows x 128 bytes on their way out, swizzled
  static constexpr int kSmem = kOffStage + 8 * 4096;
  static constexpr int kColO = 256;
  static_assert(kSmem + 1024 <= 232448, "shared memory of one CTA, static part included");
};

// Key tiles of the item that subtile s works on, as a count from it.k0.
__device__ __forceinline__ int subtile_tiles(const PagedAttnParams& p, const WorkItem& it, int s) {
  if (it.rows <= 128 * s) return 0;
  const int64_t rows = min((int64_t)it.t * kPtM + 128 * (s + 1), (int64_t)it.x.n_new * p.group);
  const int n = key_tiles<kPtKT>(visible_keys(it.x, (int)p.by_group.div((uint32_t)(rows - 1))));
  return max(0, min(n, it.k1) - it.k0);
}

template <int D, typename T>
__global__ void __launch_bounds__(kPtThreads, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                const __grid_constant__ CUtensorMap tmO, const __grid_constant__ PagedAttnParams p, const WorkPartials w, int least,
                uint32_t slope, int is_bf16, int q_vec, int q_box, int o_vec, int o_box, int box_rows) {
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
                 bar_p0 = bar0 + 160, bar_o0 = bar0 + 176, bar_tail0 = bar0 + 256;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem_raw + Cfg::kOffBar + 192);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem_raw + Cfg::kOffBar + 196);
  volatile uint32_t* masks = reinterpret_cast<volatile uint32_t*>(smem_raw + Cfg::kOffMask);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) { mbar_init(bar_full0 + 8 * i, 4); mbar_init(bar_empty0 + 8 * i, 1); mbar_init(bar_tail0 + 8 * i, 4); }
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
  const WorkShare share = find_share<kPtM, kPtKT, kPtFixed, kPtNear>(p, least, slope, false);
  publish_share(share, w);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  WorkIter<kPtM, kPtKT> iter;
  iter.start(share);
  WorkItem it;

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPtRegsLess));
  if (warp < 12) {
    // ------------------------------------------------------------- loaders --
    const int lw = warp - 8;
    uint32_t pend0 = 0, pend1 = 0;                       // barriers of the copy groups in flight, oldest first
    auto announce = [&](uint32_t bar) {                  // the copies have landed: make them visible to the MMA
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    auto push = [&](uint32_t bar) {
      copy_commit();
      if (pend0) {
        copy_wait<2>();
        announce(pend0);
      }
      pend0 = pend1;
      pend1 = bar;
    };
    auto drain = [&]() {
      copy_wait<0>();
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
      for (int i0 = 0; i0 < C; i0 += 8) {                // the exchanges first: one after the other with the copies they take 60 cycles each
        int64_t o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(0xffffffffu, off, ((i0 + i) * 32 + lane) / C);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int c = ((i0 + i) * 32 + lane) % C, row = lw * 32 + ((i0 + i) * 32 + lane) / C;
          copy16_async(dst + (c >> 3) * 16384 + row * 128 + (((c & 7) ^ (row & 7)) << 4), src + (o[i] >= 0 ? o[i] + c * 8 : 0), o[i] >= 0 ? 16 : 0);
        }
      }
    };
    // Boxes of a tile that comes by TMA: lane i of this warp knows the page of box i * 4 + lw.
    const int box = lane * 4 + lw, boxes = box_rows > 0 ? (kPtKT / box_rows - lw + 3) / 4 : 0;
    bool ok = true;
    for (int tn = 0; ok && iter.next(p, it); ++tn) {
      const int n = max(subtile_tiles(p, it, 0), subtile_tiles(p, it, 1));
      if (n == 0) { --tn; continue; }                    // no key: the softmax warps write zeros
      const int32_t* table = p.tables + (int64_t)it.r * p.width;
      // This lane's page of a tile (its box's or its row's) and the first row there.
      auto key_at = [&](int kt) { return (int)((uint32_t)kt * kPtKT + (box_rows > 0 ? box * box_rows : lw * 32 + lane)); };
      auto page_at = [&](int kt) {
        if (kt >= it.k0 + n || (box_rows > 0 && lane >= boxes)) return -1;
        const int key = key_at(kt);
        return key < it.keys ? table[p.page.div((uint32_t)key)] : -1;
      };
      auto there = [&](int page) {
        if ((unsigned)page < (unsigned)p.n_pages) return true;
        if (p.flag) atomicMax(p.flag, kPagedFlag);
        return false;
      };
      // One ring slot: the tile's keys or values, page: as page_at said.
      auto load = [&](const CUtensorMap* map, const T* pool, int kt, int page, bool keys) -> bool {
        const int slot = used % kRing, valid = it.keys - kt * kPtKT;       // rows of the tile before the last key
        const uint32_t full = bar_full0 + 8 * slot, dst = base + Cfg::kOffRing + slot * Cfg::kTile;
        if (!wait_for(bar_empty0 + 8 * slot, ((used / kRing) & 1) ^ 1u)) return false;
        ++used;
        const int key = key_at(kt);
        const int in_page = key - (int)(p.page.div((uint32_t)key) * p.page.d);
        volatile uint32_t* mask = masks + (tiles & 15) * 4;
        if (keys) ++tiles;
        if (box_rows > 0) {
          // values behind the last key: the tile is handed over by the warps that clear them
          const uint32_t landed = !keys && valid < kPtKT ? bar_tail0 + 8 * slot : full;
          if (keys) {
            const uint32_t fine = __ballot_sync(0xffffffffu, lane >= boxes || key >= it.keys || there(page));
            if (lane == 0) mask[lw] = fine;              // bit i: box i * 4 + lw
          }
          __syncwarp();
          if (lane == 0) {
            if (boxes > 0) mbar_expect_tx(landed, boxes * box_rows * D * 2);
            else mbar_arrive(landed);
          }
#pragma unroll 1
          for (int i = 0; i < boxes; ++i) {
            const int id = __shfl_sync(0xffffffffu, page, i), row = __shfl_sync(0xffffffffu, in_page, i);
            if (lane == 0) {
#pragma unroll
              for (int c = 0; c < Cfg::kChunks; ++c)
                tma_load_4d(dst + c * 16384 + (i * 4 + lw) * box_rows * 128, map, landed, c * 64, row, it.hk, id);
            }
          }
          __syncwarp();
          return true;
        }
        const int64_t off = key < it.keys && there(page) ? (int64_t)page * p.sc.b + (int64_t)in_page * p.sc.s + (int64_t)it.hk * p.sc.h : -1;
        if (keys) {
          const uint32_t m = __ballot_sync(0xffffffffu, off >= 0);
          if (lane == 0) mask[lw] = m;
        }
        copy_rows(dst, pool, off);
        push(full);
        return true;
      };
      // Pages of the tile whose values are next, of the one behind it and of the one behind that.
      int page = page_at(it.k0), next = page_at(it.k0 + 1), later = -1;
      // in the order of use: K0, then K1 V0 K2 V1 ... and the last values (one place in the code that queues a tile)
#pragma unroll 1
      for (int u = 0; u < 2 * n; ++u) {
        const bool last = u == 2 * n - 1, keys = u == 0 || ((u & 1) && !last);
        const int kt = it.k0 + (keys ? (u + 1) / 2 : last ? n - 1 : u / 2 - 1);
        if (!(ok = load(keys ? &tmK : &tmV, (const T*)(keys ? p.kp : p.vp), kt, u > 0 && keys ? next : page, keys))) break;
        if (!keys) { page = next; next = later; }
        else if (u > 0) later = page_at(kt + 1);
        if (!q_box && (u == 2 || (last && u == 1))) drain();             // the queries are on their way since before this tile's values
        if (u > 0) continue;
        // queries, once the last score MMA of the item before has read them
        if (tn > 0 && !(ok = wait_for(bar_qfree, (tn - 1) & 1))) break;
        if (q_box) {
          if (lw == 0 && lane == 0) {
            const int halves = it.rows > 128 ? 2 : 1;
            mbar_expect_tx(bar_q, halves * Cfg::kTile);
#pragma unroll 1
            for (int s = 0; s < halves; ++s)
              for (int c = 0; c < Cfg::kChunks; ++c)
                tma_load_3d(base + s * Cfg::kTile + c * 16384, &tmQ, bar_q, c * 64, it.hk * p.group,
                            it.x.q0 + (int)p.by_group.div((uint32_t)(it.t * kPtM + s * 128)));
          } else if (lane == 0) mbar_arrive(bar_q);
          __syncwarp();
        } else {
#pragma unroll 1
          for (int s = 0; s < 2; ++s) {
            const int row = s * 128 + lw * 32 + lane;
            int token, h;
            row_of<kPtM>(p, it, row, token, h);
            const int64_t q = row < it.rows ? (int64_t)(it.x.q0 + token) * p.sq.s + (int64_t)h * p.sq.h : -1;
            const uint32_t dst = base + s * Cfg::kTile;
            if (q_vec) copy_rows(dst, (const T*)p.q, q);
            else {                                           // rows at any address: element by element
#pragma unroll 1
              for (int c = 0; c < D; ++c) {
                const int r = lw * 32 + lane;
                T* to = reinterpret_cast<T*>(smem_raw + s * Cfg::kTile + (c >> 6) * 16384 + r * 128 + ((((c >> 3) & 7) ^ (r & 7)) << 4)) + (c & 7);
                *to = q >= 0 ? ((const T*)p.q)[q + c] : from_f<T>(0.f);
              }
            }
          }
          push(bar_q);
        }
      }
      if (!ok) break;
    }
    drain();
  } else if (warp > 12) {
    // ------------------------------------------------------------ clearing --
    int used = 0;                                        // ring slots so far
    uint32_t cleared = 0;                                // by slot: parity of the tiles cleared there
    while (box_rows > 0 && iter.next(p, it)) {
      const int n = max(subtile_tiles(p, it, 0), subtile_tiles(p, it, 1));
      if (n == 0) continue;
      used += 2 * n;
      const int slot = (used - 1) % kRing, valid = it.keys - (it.k0 + n - 1) * kPtKT;   // the item's last values
      if (valid >= kPtKT) continue;
      if (!__all_sync(0xffffffffu, mbar_wait(bar_tail0 + 8 * slot, (cleared >> slot) & 1, abort_flag))) break;
      cleared ^= 1u << slot;
      uint8_t* rows = smem_raw + Cfg::kOffRing + slot * Cfg::kTile;
#pragma unroll 1
      for (int i = (warp - 13) * 32 + lane; i < (kPtKT - valid) * Cfg::kChunks * 8; i += 96) {
        const int row = valid + i / (Cfg::kChunks * 8), c = i % (Cfg::kChunks * 8);
        *reinterpret_cast<uint4*>(rows + (c >> 3) * 16384 + row * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {                                   // four arrivals from three warps
        mbar_arrive(bar_full0 + 8 * slot);
        if (warp == 15) mbar_arrive(bar_full0 + 8 * slot);
      }
    }
  } else if (warp == 12) {
    // ---------------------------------------------------------- MMA issuer --
    // The whole warp walks the loop and one lane issues: counts and addresses are the same in all lanes, so that descriptors
    // are formed on the uniform datapath. (Formed by a thread of its own, the 32 products of a
    // step took 4500 cycles to issue, twice the time they take to run.)
    const bool leader = elect_one();
    const uint32_t idesc_s = idesc_f16(is_bf16, 0, 0, 128, 128);
    const uint32_t idesc_o = idesc_f16(is_bf16, 0, 1, 128, D);
    // descriptors of Q_A and of ring slot 0; the others are offsets (in 16-byte units) from these
    const uint64_t dq = smem_desc_sw128(base, 16, 1024), dk0 = smem_desc_sw128(base + Cfg::kOffRing, 16, 1024),
                   dv0 = smem_desc_sw128(base + Cfg::kOffRing, 16384, 1024);
    int used = 0, np[2] = {0, 0};                        // ring slots taken; weight tiles awaited per subtile
    auto wait_full = [&](int u) { return mbar_wait(bar_full0 + 8 * (u % kRing), (u / kRing) & 1, abort_flag); };
    auto issue_s = [&](int s, int slot) {                // by the leader
#pragma unroll
      for (int c = 0; c < Cfg::kChunks; ++c) {
        uint64_t a[4], b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          a[k] = dq + (uint32_t)((s * Cfg::kTile + c * 16384 + k * 32) >> 4);
          b[k] = dk0 + (uint32_t)((slot * Cfg::kTile + c * 16384 + k * 32) >> 4);
        }
        umma_f16_x4(tmem_base + 128 * s, a, b, idesc_s, c > 0 ? 1u : 0u);
      }
      umma_commit(bar_s0 + 8 * s);
    };
    bool ok = true;
    for (int tn = 0; ok && iter.next(p, it); ++tn) {
      const int count[2] = {__shfl_sync(0xffffffffu, subtile_tiles(p, it, 0), 0), __shfl_sync(0xffffffffu, subtile_tiles(p, it, 1), 0)};
      const int n = max(count[0], count[1]);
      if (n == 0) { --tn; continue; }
      int uk = used++;                                   // slot of the next key tile
      if (!__all_sync(0xffffffffu, wait_full(uk) && mbar_wait(bar_q, tn & 1, abort_flag))) break;
      tc_fence_after();
      if (leader) {
        if (count[0] > 0) issue_s(0, uk % kRing);
        if (count[1] > 0) issue_s(1, uk % kRing);
        umma_commit(bar_empty0 + 8 * (uk % kRing));
        if (n == 1) umma_commit(bar_qfree);
      }
      __syncwarp();
#pragma unroll 1
      for (int i = 0; i < n; ++i) {
        const bool more = i + 1 < n;
        if (more) uk = used++;
        const int uv = used++;
        if (!__all_sync(0xffffffffu, (!more || wait_full(uk)) && wait_full(uv))) { ok = false; break; }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (i >= count[s]) continue;
          if (!__all_sync(0xffffffffu, mbar_wait(bar_p0 + 8 * s, np[s] & 1, abort_flag))) { ok = false; break; }
          ++np[s];
          tc_fence_after();
          if (leader) {
            uint64_t b[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) b[k] = dv0 + (uint32_t)(((uv % kRing) * Cfg::kTile + k * 2048) >> 4);
            umma_f16_ts_x8(tmem_base + Cfg::kColO + D * s, tmem_base + 128 * s, b, idesc_o, i > 0 ? 1u : 0u);
            if (i + 1 < count[s]) issue_s(s, uk % kRing);
            else umma_commit(bar_o0 + 8 * s);            // the subtile's last product
          }
          __syncwarp();
        }
        if (!ok) break;
        if (leader) {
          umma_commit(bar_empty0 + 8 * (uv % kRing));
          if (more) {
            umma_commit(bar_empty0 + 8 * (uk % kRing));
            if (i + 2 == n) umma_commit(bar_qfree);      // the item's last score MMA
          }
        }
        __syncwarp();
      }
    }
    // the last commit signals shared memory: not after the CTA is gone
    if (used > 0) mbar_wait(bar_empty0 + 8 * ((used - 1) % kRing), ((used - 1) / kRing) & 1, abort_flag);
  }
  } else {
    // ------------------------------------------------------------- softmax --
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPtRegsMore));
    const int sub = warp >> 2, qtr = warp & 3;
    const int row = sub * 128 + qtr * 32 + lane;         // of the item
    const uint32_t lanes = (uint32_t)(qtr * 32) << 16;
    const uint32_t tmem_s = tmem_base + 128 * sub + lanes, tmem_o = tmem_base + Cfg::kColO + D * sub + lanes;
    int ns = 0, no = 0, tiles = 0;                       // score tiles and items of this subtile so far; key tiles so far
    bool ok = true, again = false;                       // again: an output is NaN or infinite
    while (ok && iter.next(p, it)) {
      const int count = subtile_tiles(p, it, sub), n = max(count, subtile_tiles(p, it, sub ^ 1));
      int token, h;
      row_of<kPtM>(p, it, row, token, h);
      const bool real = row < it.rows, busy = it.rows > sub * 128 + qtr * 32;
      const int lim = real ? visible_keys(it.x, token) : INT32_MAX;
      const int lim_min = __reduce_min_sync(0xffffffffu, lim);
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int i = 0; i < count; ++i) {
        const int key0 = (it.k0 + i) * kPtKT;
        if (!__all_sync(0xffffffffu, mbar_wait(bar_s0 + 8 * sub, ns & 1, abort_flag))) { ok = false; break; }
        ++ns;
        tc_fence_after();
        if (!busy) {                                     // no row in this warp: whatever stands in P reaches no other row
          if (lane == 0) mbar_arrive(bar_p0 + 8 * sub);
          continue;
        }
        volatile const uint32_t* mask = masks + ((tiles + i) & 15) * 4;
        const bool all = (mask[0] & mask[1] & mask[2] & mask[3]) == 0xffffffffu;
        if (!all || key0 > lim_min - kPtKT) {
          // What a row does not see becomes -inf where it lies, in pieces: rare tiles take longer, the others have no code for it.
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            const int left = lim - key0 - 32 * c;        // columns of this piece that the row sees
            uint32_t bits = left >= 32 ? 0xffffffffu : left <= 0 ? 0u : (1u << left) - 1;
            if (!all) {
              if (box_rows > 0) {
#pragma unroll 1
                for (int e = 0; e < 32; ++e) {
                  const int at = (32 * c + e) / box_rows;
                  if (!((mask[at & 3] >> (at >> 2)) & 1)) bits &= ~(1u << e);
                }
              } else bits &= mask[c];
            }
            if (__all_sync(0xffffffffu, bits == 0xffffffffu)) continue;
            uint32_t x[32];
            tmem_ld32(tmem_s + 32 * c, x);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) if (!((bits >> e) & 1)) x[e] = 0xff800000u;
            tmem_st32(tmem_s + 32 * c, x);
          }
          tmem_st_wait();
        }
        uint32_t r[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(tmem_s + 32 * c, r + 32 * c);
        tmem_ld_wait();
        float x0 = -INFINITY, x1 = -INFINITY, x2 = -INFINITY, x3 = -INFINITY;
#pragma unroll
        for (int e = 0; e < 128; e += 8) {
          x0 = max3(x0, __uint_as_float(r[e]), __uint_as_float(r[e + 1]));
          x1 = max3(x1, __uint_as_float(r[e + 2]), __uint_as_float(r[e + 3]));
          x2 = max3(x2, __uint_as_float(r[e + 4]), __uint_as_float(r[e + 5]));
          x3 = max3(x3, __uint_as_float(r[e + 6]), __uint_as_float(r[e + 7]));
        }
        const float top = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3)) * p.scale_log2;
        const bool move = top > m && (m == -INFINITY || top - m > 8.f);
        if (__any_sync(0xffffffffu, move)) {
          const float c = !move ? 1.f : m == -INFINITY ? 0.f : ex2_approx(m - top);
          if (move) { m = top; l *= c; }
          if (i > 0) {                                   // these scores were issued behind the last product into O
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              uint32_t o[16];
              tmem_ld16(tmem_o + d, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * c);
              tmem_st16(tmem_o + d, o);
            }
          }
        }
        const float sub_m = m == -INFINITY ? 0.f : m;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float p0 = ex2_approx(fmaf(__uint_as_float(r[32 * c + 2 * e]), p.scale_log2, -sub_m));
            const float p1 = ex2_approx(fmaf(__uint_as_float(r[32 * c + 2 * e + 1]), p.scale_log2, -sub_m));
            l0 += p0;
            l1 += p1;
            pk[e] = pack2<T>(p0, p1);
          }
          tmem_st16(tmem_s + 16 * c, pk);                // over the scores
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
      float odd = 0.f;                                   // NaN once an output is NaN or infinite
      if (busy) {
        // Rows leave through the warp's staging buffer (swizzled), 128 bytes of each at a time and as one copy for all 32:
        // partial results as they lie there (the joining kernel reads them so), outputs through a tensor map
        // where all 32 rows are the item's and the heads of the group divide 32, else by eight lanes per row. (A thread storing its own
        // row piece by piece touched 32 lines per store: 8000 cycles per item; eight lanes per row take 5000.)
        uint8_t* stage = smem_raw + Cfg::kOffStage + warp * 4096;
        const int64_t o_row = real ? (int64_t)(it.x.q0 + token) * p.so.s + (int64_t)h * p.so.h : -1;
        const bool boxed = o_box && it.rows >= sub * 128 + qtr * 32 + 32;
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
          if (slot >= 0 || !(d & 32)) {                  // the buffer's last copy has read it
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
          }
          if (slot >= 0) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(r[4 * c], r[4 * c + 1], r[4 * c + 2], r[4 * c + 3]);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              bulk_store_1d(w.o + partial_at<D>(slot, sub * 128 + qtr * 32, d), smem_u32(stage), 4096);
              bulk_commit();
            }
            continue;
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) { v[u] = __uint_as_float(r[8 * c + u]) * inv; odd = fmaf(v[u], 0.f, odd); }
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((((d & 32) / 8 + c) ^ (lane & 7)) << 4)) =
                make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
            if (!o_vec && real)                          // rows at any address
#pragma unroll
              for (int u = 0; u < 8; ++u) ((T*)p.o)[o_row + d + 8 * c + u] = from_f<T>(v[u]);
          }
          if (!o_vec || !(d & 32)) continue;
          if (boxed) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&tmO, smem_u32(stage), d - 32, it.hk * p.group, it.x.q0 + token);
              bulk_commit();
            }
            continue;
          }
          __syncwarp();
#pragma unroll 2
          for (int j = 0; j < 8; ++j) {
            const int rr = j * 4 + (lane >> 3), c = lane & 7;
            const uint4 v = *reinterpret_cast<const uint4*>(stage + rr * 128 + ((c ^ (rr & 7)) << 4));
            const int64_t at = __shfl_sync(0xffffffffu, o_row, rr);
            if (at >= 0) *reinterpret_cast<uint4*>((T*)p.o + at + d - 32 + c * 8) = v;
          }
          __syncwarp();
        }
        if (slot >= 0 && real)
          *reinterpret_cast<float2*>(w.ml + ((int64_t)slot * kPtM + row) * 2) = make_float2(m, l);
        again |= __any_sync(0xffffffffu, slot < 0 && real && isnan(odd));
      }
      tc_fence_before();                                 // O is read: the next item's weights may follow
    }
    if (lane == 0) bulk_wait_all<0>();                   // the copies must be done with shared memory before the CTA exits
    __syncwarp();
    // Rows that came out as NaN or infinite once more, now that nobody waits for this warp: a row takes 0.6 us per key, 32 rows of
    // 110,000 keys more than the two seconds after which the other warps' waits end.
    if (again && ok) {
      iter.start(WorkShare{iter.last[-1], iter.last, 0});
      while (iter.next(p, it)) {
        if (partial_slot(it) >= 0) continue;             // the joining kernel's
        const int first = sub * 128 + qtr * 32, last = min(first + 32, it.rows);
#pragma unroll 1
        for (int row = first; row < last; ++row) {
          int token, h;
          row_of<kPtM>(p, it, row, token, h);
          const T* o = (const T*)p.o + (int64_t)(it.x.q0 + token) * p.so.s + (int64_t)h * p.so.h;
          bool odd = false;
#pragma unroll
          for (int d = 0; d < D; d += 32) odd |= !isfinite(to_f(__ldcg(o + d + lane)));
          if (__any_sync(0xffffffffu, odd)) paged_row_plain<T, D>(p, it.x, it.r, token, h);
        }
      }
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
  TempBuf part(partial_bytes(grid, kPtM, D), st, Scratch::kOwnPool);
  if (!part.ok()) return MT_ERR_CUDA;
  const WorkPartials w = partials_in(part.ptr, grid, kPtM, D);
  auto vec = [](const void* x, mt_strides3 s) { return aligned16(x) && s.h % 8 == 0 && s.s % 8 == 0; };
  const int bf16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap tq{}, tk{}, tv{}, to{};
  int rc;
  // pages as boxes of a tensor map {head_dim, row, head, page}, whose strides are multiples of one another
  const int64_t page = p.page.d, fits = page % 128 == 0 ? 128 : page & -page;   // largest power of two in page: a box never leaves its page
  int box_rows = 0;
  if (fits >= 8 && p.sc.s > 0 && p.sc.h > 0 && p.sc.b > 0 && p.sc.h % p.sc.s == 0 && p.sc.b % p.sc.h == 0 && p.sc.b < (1ll << 38) &&
      p.n_pages > 0) {
    box_rows = fits < 128 ? (int)fits : 128;
    const uint64_t dims[4] = {(uint64_t)D, (uint64_t)page, (uint64_t)p.kv_heads, (uint64_t)p.n_pages};
    const uint64_t strides[3] = {(uint64_t)p.sc.s, (uint64_t)p.sc.h, (uint64_t)p.sc.b};
    const uint32_t box[4] = {64, (uint32_t)box_rows, 1, 1};
    if ((rc = make_tmap_nd(&tk, p.kp, bf16, 4, dims, strides, box))) return rc;
    if ((rc = make_tmap_nd(&tv, p.vp, bf16, 4, dims, strides, box))) return rc;
  }
  // query and output rows as boxes {head_dim, heads of a group, tokens} of 128 and 32 rows
  auto rows_map = [&](CUtensorMap* m, int* on, const void* x, mt_strides3 s, int rows) {
    *on = vec(x, s) && rows % p.group == 0 && s.h > 0 && s.s > 0 && s.s % s.h == 0 && s.s < (1ll << 38);
    if (!*on) return (int)MT_OK;
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)p.heads, (uint64_t)p.rows};
    const uint64_t strides[2] = {(uint64_t)s.h, (uint64_t)s.s};
    const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)(rows / p.group)};
    return make_tmap_nd(m, x, bf16, 3, dims, strides, box);
  };
  int q_box, o_box;
  if ((rc = rows_map(&tq, &q_box, p.q, p.sq, 128)) || (rc = rows_map(&to, &o_box, p.o, p.so, 32))) return rc;
  MT_CHECK_CUDA(launch_overlapped(kern, dim3((unsigned)grid), dim3(kPtThreads), Cfg::kSmem, st, tq, tk, tv, to, p, w, 3,
                                  tile_slope<kPtM, kPtKT>(p.group), bf16, vec(p.q, p.sq), q_box, vec(p.o, p.so), o_box, box_rows));
  count_launch();
  return launch_join<T, D, kPtM, kPtKT>(p, w, grid, st);
}

int attn_paged_tc(const PagedAttnParams& p, int head_dim, int dtype, cudaStream_t st) {
  if (dtype == MT_F16) return head_dim == 64 ? launch_paged_tc<64, __half>(p, st) : launch_paged_tc<128, __half>(p, st);
  return head_dim == 64 ? launch_paged_tc<64, __nv_bfloat16>(p, st) : launch_paged_tc<128, __nv_bfloat16>(p, st);
}

}  // namespace mt
