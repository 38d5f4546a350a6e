// Launches of the matrix-core attention over a paged KV cache (paged_attn_mfma.hpp).
#include "paged_attn_mfma.hpp"

namespace mi {

PagedPlan paged_plan(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t seq_len,
                     int64_t head_dim, int32_t dtype, int64_t num_splits) {
  PagedPlan p{};
  p.mfma = head_dim == 64 || head_dim == 128 || head_dim == 256;
  if (!p.mfma) return p;
  const int64_t n = seq_len * (n_heads / n_kv_heads);
  // 2 tiles a block where one does not hold all rows and the registers hold two: each key
  // is read and widened half as often (511 tokens over 4096 keys, head_dim 64: 47 us, 54 with
  // one tile and 53 with four, whose registers leave one wave a SIMD)
  p.r = n <= 16 || head_dim > (dtype == MI_DTYPE_F32 ? 64 : 128) ? 1 : 2;
  p.tiles = (n + 16 * p.r - 1) / (16 * p.r);
  p.parts = num_splits <= 1 ? 0 : num_splits;
  return p;
}

int64_t paged_mfma_splits(const PagedPlan& plan, int64_t batch, int64_t n_kv_heads,
                          int64_t head_dim, int64_t units, int64_t entry_bytes) {
  // blocks of 4 waves that are resident at once, by their registers (of a CU's 3, 2 and 1; one
  // more each, in us: 64 rows of up to 4096 keys, head_dim 64, 39.0, 46.2 with 4; 64 rows of up
  // to 8192, 128, 123.0, 136.3 with 3; 1 row of 60000, 256, 54.7, 60.6 with 2)
  const int64_t fill = (head_dim == 64 && plan.r == 1 ? 3 : head_dim == 256 ? 1 : 2) *
                       (int64_t)device_cu_count();
  const int64_t blocks = n_kv_heads * plan.tiles;
  // a block a row, and one launch, where no row has more than 16 units of keys, or 32 of 64
  // bytes (us, calls among others, undivided and divided; 2000 8-bit keys of 64 dims: 1 row
  // 12.3 and 16.2, 16 rows 11.2 and 15.9, 64 rows 19.3 and 26.2, 3000 keys 16.8 and 16.0, 17.7
  // and 17.6, 27.0 and 31.2; bf16 keys of 128 dims, 800: 17.0 and 15.8, 17.5 and 22.1, 31.8 and
  // 35.5, 1500: 25.8 and 16.5, 27.1 and 22.8, 52.4 and 43.7)
  const int64_t most_units = head_dim * entry_bytes <= 64 ? 32 : 16;
  if (units <= most_units) return 1;
  int64_t parts = fill / blocks;
  const int64_t most = batch * ((units + 3) / 4);
  if (parts > most) parts = most;
  return parts < 1 ? 1 : parts;
}

int64_t paged_mfma_workspace(const PagedPlan& plan, int64_t n_kv_heads, int64_t head_dim) {
  return n_kv_heads * plan.tiles * plan.parts * 2 * (16 * plan.r) * (head_dim + 2);
}

namespace {

template <typename T, bool E8, int D, int R>
void launch_tiles(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
  const dim3 grid((unsigned)(a.Hkv * (p.parts > a.B ? p.parts : a.B)), (unsigned)p.tiles);
  if (p.tiles == 1)
    hipLaunchKernelGGL((paged_attn_mfma_kernel<T, E8, D, R, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_attn_mfma_kernel<T, E8, D, R, false>), grid, dim3(256), 0, st, a);
  if (p.parts > 0) {
    const int64_t blocks = (int64_t)a.B * a.Hkv * p.tiles;
    // rows of a tile apart where their tiles alone are fewer than the compute units (16 rows of
    // up to 8192 keys, 8 KV heads: 62.7 us in all, 64.1 together; 1 row of 131072 56.1 and 60.2)
    const unsigned apart = blocks < device_cu_count() ? (unsigned)a.kv_rows : 1u;
    hipLaunchKernelGGL((paged_mfma_join_kernel<T, D>), dim3((unsigned)blocks, apart), dim3(256), 0,
                       st, a);
  }
}

template <typename T, bool E8>
void launch_128(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (p.r == 2) return launch_tiles<T, E8, 128, 2>(a, p, st);
  }
  launch_tiles<T, E8, 128, 1>(a, p, st);
}

template <typename T, bool E8>
void launch(const PagedAttnArgs& a, const PagedPlan& p, hipStream_t st) {
  if (a.D == 64)
    p.r == 1 ? launch_tiles<T, E8, 64, 1>(a, p, st) : launch_tiles<T, E8, 64, 2>(a, p, st);
  else if (a.D == 128)
    launch_128<T, E8>(a, p, st);
  else
    launch_tiles<T, E8, 256, 1>(a, p, st);
}

}  // namespace

void paged_attn_mfma_launch(const PagedAttnArgs& a, const PagedPlan& plan, int32_t dtype, bool e8,
                            hipStream_t st) {
  if (dtype == MI_DTYPE_BF16)
    e8 ? launch<bf16_t, true>(a, plan, st) : launch<bf16_t, false>(a, plan, st);
  else if (dtype == MI_DTYPE_F32)
    e8 ? launch<float, true>(a, plan, st) : launch<float, false>(a, plan, st);
  else
    e8 ? launch<f16_t, true>(a, plan, st) : launch<f16_t, false>(a, plan, st);
}

}  // namespace mi
