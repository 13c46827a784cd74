// Attention of every request's new rows over the pages of its key/value cache (mt_attn_paged).
#include "paged.cuh"

namespace mt {

// One output row (a token's head) by one warp, straight from the definition: lane l holds D/32
// neighbouring elements of q and o, scores are fp32 dot products, and only the visible keys are touched.
template <typename T, int D>
__device__ __forceinline__ void paged_row_plain(const PagedAttnParams& p, const PagedRequest& x, int r, int i, int h) {
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
  T* op = (T*)p.o + (int64_t)(x.q0 + i) * p.so.s + (int64_t)h * p.so.h + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = from_f<T>(l == 0.f ? 0.f : o[e] / l);
}

template <typename T, int D>
__global__ void __launch_bounds__(128)
paged_plain_kernel(const PagedAttnParams p) {
  const int64_t at = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int token = (int)(at / p.heads), h = (int)(at % p.heads);
  if (token >= p.rows || token < p.starts[0] || token >= p.starts[p.requests]) return;
  int lo = 0, hi = p.requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid] <= token) lo = mid; else hi = mid;
  }
  const PagedRequest x = paged_request(p, lo);
  if (token - x.q0 < x.n_new) paged_row_plain<T, D>(p, x, lo, token - x.q0, h);
}

template <typename T, int D>
static int launch_plain(const PagedAttnParams& p, cudaStream_t st) {
  const int64_t warps = (int64_t)p.rows * p.heads;
  paged_plain_kernel<T, D><<<(unsigned)((warps + 3) / 4), 128, 0, st>>>(p);
  MT_LAUNCH_CHECK();
  return MT_OK;
}

}  // namespace mt

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
  MT_REQUIRE(requests <= (1 << 20) && rows * heads < (1ll << 31) && max_new >= 0, "attn_paged: too many query rows");
  const int64_t unit = 16 / (int64_t)dtype_size(dtype);
  MT_REQUIRE(spages.b % unit == 0 && spages.h % unit == 0 && spages.s % unit == 0 && aligned16(k_pages) && aligned16(v_pages),
             "attn_paged: the rows of the pools must be 16-byte aligned");
  MT_REQUIRE(scale > 0.f && scale <= 3.4028235e38f, "attn_paged: scale must be a positive finite number");
  if (requests == 0 || rows == 0) return MT_OK;
  PagedAttnParams p{};
  p.q = q; p.kp = k_pages; p.vp = v_pages; p.o = o;
  p.sq = sq; p.sc = spages; p.so = so;
  p.tables = tables; p.starts = starts; p.kv_len = kv_len;
  p.requests = (int)requests; p.width = (int)width; p.rows = (int)rows; p.heads = (int)heads; p.kv_heads = (int)kv_heads;
  p.group = (int)(heads / kv_heads); p.n_pages = (int)n_pages;
  p.page = FastDiv((uint32_t)page_size); p.by_group = FastDiv((uint32_t)p.group);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.flag = device_flag_ptr();
  cudaStream_t st = as_stream(stream);
  MT_DISPATCH_FLOAT(dtype, T, return head_dim == 64 ? (launch_plain<T, 64>(p, st)) : (launch_plain<T, 128>(p, st)));
  return MT_OK;
}

}  // extern "C"
