// C entry point of attention over pages: argument checks and the choice of the kernel, by the rows (new tokens times the query
// heads of the group) that the caller expects per key/value head.
#include "attention_paged.cuh"

using namespace mt;

extern "C" {

int mt_attn_paged(const void* q, const void* k_pages, const void* v_pages, void* o, mt_strides3 sq, mt_strides3 spages,
                  mt_strides3 so, const int32_t* tables, const int32_t* starts, const int32_t* kv_len, int64_t requests,
                  int64_t width, int64_t rows, int64_t max_new, int64_t heads, int64_t kv_heads, int64_t head_dim,
                  int64_t page_size, int64_t n_pages, float scale, int dtype, void* stream) {
  MT_REQUIRE(q && k_pages && v_pages && o && tables && starts && kv_len && requests >= 0 && rows >= 0 && heads > 0,
             "attn_paged: bad arguments");
  MT_REQUIRE(dtype == MT_F32 || dtype == MT_F16 || dtype == MT_BF16, "attn_paged: unsupported dtype code %d", dtype);
  MT_REQUIRE(kv_heads > 0 && heads % kv_heads == 0, "attn_paged: query heads must be a multiple of key/value heads");
  MT_REQUIRE(head_dim == 64 || head_dim == 128, "attn_paged: head_dim must be 64 or 128");
  MT_REQUIRE(width >= 1 && width < (1ll << 31) && page_size >= 1 && page_size < (1ll << 30) && width * page_size < (1ll << 31) && n_pages >= 0 &&
             n_pages < (1ll << 31), "attn_paged: a table row has to span between 1 and 2^31 - 1 positions");
  MT_REQUIRE(requests <= (1 << 20) && rows < (1ll << 28) && heads < (1ll << 28) && rows * heads < (1ll << 28) && max_new >= 0, "attn_paged: too many query rows");
  const int64_t unit = 16 / (int64_t)dtype_size(dtype);
  MT_REQUIRE(spages.b % unit == 0 && spages.h % unit == 0 && spages.s % unit == 0 && aligned16(k_pages) && aligned16(v_pages),
             "attn_paged: the rows of the pools must be 16-byte aligned");
  MT_REQUIRE(sq.h >= 0 && sq.s >= 0 && so.h >= 0 && so.s >= 0 && spages.b >= 0 && spages.h >= 0 && spages.s >= 0,
             "attn_paged: negative strides");      // an offset below 0 is a row that is not there
  MT_REQUIRE(o != q, "attn_paged: the output needs a buffer of its own");
  MT_REQUIRE(scale > 0.f && scale < 2e38f, "attn_paged: scale must be a positive finite number");
  if (requests == 0 || rows == 0) return MT_OK;
  PagedAttnParams p{};
  p.q = q; p.kp = k_pages; p.vp = v_pages; p.o = o;
  p.sq = sq; p.sc = spages; p.so = so;
  p.tables = tables; p.starts = starts; p.kv_len = kv_len;
  p.requests = (int)requests; p.width = (int)width; p.rows = (int)rows; p.heads = (int)heads; p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads); p.n_pages = (int)n_pages;
  p.page = FastDiv((uint32_t)page_size); p.by_group = FastDiv((uint32_t)p.group);
  p.scale_log2 = scale * 1.4426950408889634f;
  auto on = [&](const void* x, mt_strides3 t, int64_t elems) {
    return (uintptr_t)x % (elems * dtype_size(dtype)) == 0 && t.h % elems == 0 && t.s % elems == 0;
  };
  p.q_pairs = on(q, sq, 2);
  p.o_quads = on(o, so, 4);
  p.flag = device_flag_ptr();
  cudaStream_t st = as_stream(stream);
  const int64_t row_hint = (max_new < rows ? max_new : rows) * p.group;
  const int few = dtype == MT_F32 ? 8 : 32;
  p.most_rows = INT32_MAX;
  if (row_hint <= few) return attn_paged_few(p, row_hint, (int)head_dim, dtype, st);
  // Where most requests bring much less than the largest does (a token each, say, beside pieces of prompts), those whose rows
  // fit in one small tile can go to the kernel for few rows first: a tile of many rows takes its time whatever is in it. At
  // head_dim 128 that time is about what its keys and values take to arrive, and one launch is better (24 requests, 10
  // heads: 95 us against 101; 64 requests, 10/2 heads: 72 against 81); at 64 and in fp32 it is not (64 requests, 12 heads of 64, fp16: 101 us
  // against 74 in two; 24 in fp32: 210 against 133).
  const int64_t small = few == 8 ? (p.group <= 1 ? 1 : p.group <= 2 ? 2 : p.group <= 4 ? 4 : 8) : (p.group + 7) / 8 * 8;
  if ((head_dim == 64 || dtype == MT_F32) && requests > 1 && max_new < rows && p.group <= few && 2 * rows <= requests * max_new) {
    PagedAttnParams f = p;
    f.most_rows = (int)small;
    if (int rc = attn_paged_few(f, small, (int)head_dim, dtype, st)) return rc;
    p.least_rows = (int)small + 1;
  }
  return dtype == MT_F32 ? attn_paged_f32(p, (int)head_dim, st) : attn_paged_tc(p, (int)head_dim, dtype, st);
}

}  // extern "C"
