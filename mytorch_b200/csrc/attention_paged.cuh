// Launchers of the kernels behind mt_attn_paged.
#pragma once
#include "paged.cuh"

namespace mt {
int attn_paged_few(const PagedAttnParams& p, int64_t row_hint, int head_dim, int dtype, cudaStream_t st);
int attn_paged_tc(const PagedAttnParams& p, int head_dim, int dtype, cudaStream_t st);
int attn_paged_f32(const PagedAttnParams& p, int head_dim, cudaStream_t st);
}  // namespace mt
