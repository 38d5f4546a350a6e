// Launches of the matrix-core attention over a paged KV cache (paged_attn_mfma.hpp).
#include "paged_attn_mfma.hpp"

#ifndef V_ROWS_FROM
#define V_ROWS_FROM 64
#endif
#ifndef V_PIPE1
#define V_PIPE1 false
#endif
#ifndef V_PIPE2
#define V_PIPE2 false
#endif
#ifndef V_RR
#define V_RR 2
#endif

namespace mi {

PagedPlan paged_plan(int64_t n_heads, int64_t n_kv_heads, int64_t seq_len, int64_t head_dim,
                     int32_t dtype) {
  PagedPlan p{};
  p.mfma = dtype != MI_DTYPE_F32 && head_dim % 64 == 0;
  if (!p.mfma) return p;
  const int64_t n = seq_len * (n_heads / n_kv_heads);
  p.rows = n > V_ROWS_FROM;
  p.r = n <= 16 || head_dim > 128 ? 1 : 2;
  if (p.rows && head_dim <= 128) p.r = V_RR;
  const int64_t block = (p.rows ? 64 : 16) * p.r;
  p.tiles = (n + block - 1) / block;
  return p;
}

namespace {

template <typename T, bool E8, int D>
void launch(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.B * a.Hkv * a.splits), (unsigned)p.tiles), block(256);
  if constexpr (D <= 128) {
    if (p.rows)
      hipLaunchKernelGGL((paged_attn_mfma_kernel<T, E8, D, V_RR, true, false>), grid, block, 0, st, a);
    else if (p.r == 2)
      hipLaunchKernelGGL((paged_attn_mfma_kernel<T, E8, D, 2, false, V_PIPE2>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((paged_attn_mfma_kernel<T, E8, D, 1, false, V_PIPE1>), grid, block, 0, st, a);
  } else {
    if (p.rows)
      hipLaunchKernelGGL((paged_attn_mfma_kernel<T, E8, D, 1, true, false>), grid, block, 0, st, a);
    else
      hipLaunchKernelGGL((paged_attn_mfma_kernel<T, E8, D, 1, false, false>), grid, block, 0, st, a);
  }
}

template <typename T, bool E8>
void launch_dim(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
  if (a.D == 64)
    launch<T, E8, 64>(a, p, st);
  else if (a.D == 128)
    launch<T, E8, 128>(a, p, st);
  else if (a.D == 192)
    launch<T, E8, 192>(a, p, st);
  else
    launch<T, E8, 256>(a, p, st);
}

}  // namespace

void paged_attn_mfma_launch(const PagedAttnArgs& a, const PagedPlan& plan, int32_t dtype, bool e8,
                            hipStream_t st) {
  if (dtype == MI_DTYPE_BF16)
    e8 ? launch_dim<bf16_t, true>(a, plan, st) : launch_dim<bf16_t, false>(a, plan, st);
  else
    e8 ? launch_dim<f16_t, true>(a, plan, st) : launch_dim<f16_t, false>(a, plan, st);
}

}  // namespace mi
