// Attention over a paged KV cache: what its kernels share (arguments, the work
// of a block, partial softmax states).
#pragma once

#include "paged_common.hpp"

namespace mi {

struct PagedAttnArgs {
  const void* q;
  const void* kp;           // [pages, Hkv, P, D]
  const void* vp;           // [pages, Hkv, D, P]
  const float* scales;      // [pages, Hkv, 2]: K, V (8-bit pages)
  const int32_t* table;
  const int64_t* seq_lens;
  const int64_t* lens;      // query tokens of each row; null: S
  float* part_acc;          // sums of key ranges (unnormalised): one block a (row, range):
  float* part_ml;           //   [B * Hq * S, splits, D] and [.., 2], their m and l
  void* out;
  float* lse;
  int64_t q_sb, q_sh, q_ss;
  int64_t o_sb, o_sh, o_ss;
  int64_t t_sb, num_pages;
  int32_t B, Hq, Hkv, group, S, D, P, p_shift, slots, splits;
  int32_t tiles, parts, kv_rows;   // matrix cores: see PagedPlan; query rows of a block
  float scale_log2;
  int32_t q_vec, o_vec;     // q rows 16-byte, 4 elements of out rows aligned
};

// How a call is laid on blocks.
struct PagedPlan {
  bool mfma;       // the matrix-core kernel, else one block a (query row, key range)
  int r;           // 16-row tiles of a block
  int64_t tiles;   // blocks along the query rows of a KV head
  int64_t parts;   // blocks along a KV head's keys: parts of the list of all rows' keys,
                   // or 0: one block a row (no second launch)
};
PagedPlan paged_plan(int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t seq_len,
                     int64_t head_dim, int32_t dtype, int64_t num_splits);
int64_t paged_mfma_splits(const PagedPlan& plan, int64_t batch, int64_t n_kv_heads,
                          int64_t head_dim, int64_t units, int64_t entry_bytes);
int64_t paged_mfma_workspace(const PagedPlan& plan, int64_t n_kv_heads, int64_t head_dim);
void paged_attn_mfma_launch(const PagedAttnArgs& a, const PagedPlan& plan, int32_t dtype, bool e8,
                            hipStream_t st);

// The maximum of no scores: the lowest float, so that every finite score is above it or equal,
// and not -inf, whose difference from a masked score would be a NaN.
constexpr float kLowest = -3.402823466e38f;

// Row b's keys as its query tokens see them: token s sees keys [0, vis(s)).
struct RowKeys {
  int64_t base;   // keys before the row's first query token
  int32_t n;      // query tokens that are real
  int32_t cap;    // keys that the row's slots hold
  __device__ inline int vis(int s) const {
    if (s >= n) return 0;
    const int64_t v = base + s + 1;
    return (int)(v < 0 ? 0 : (v < cap ? v : cap));
  }
};
__device__ inline RowKeys row_keys(const PagedAttnArgs& a, int b) {
  RowKeys r;
  r.cap = a.slots << a.p_shift;
  int64_t n = a.lens != nullptr ? a.lens[b] : a.S;
  n = n < 0 ? 0 : (n > a.S ? a.S : n);
  r.n = (int)n;
  // (a length far outside the slots keeps its meaning without overflowing)
  int64_t len = a.seq_lens[b];
  const int64_t most = (int64_t)r.cap + a.S;
  len = len < 0 ? 0 : (len > most ? most : len);
  r.base = len - n;
  return r;
}

// Keys [lo, hi) of `vis` that split `i` of `splits` takes: whole units of 64.
__device__ inline void split_range(int vis, int i, int splits, int* lo, int* hi) {
  const int units = (vis + 63) >> 6;
  const int per = (units + splits - 1) / splits;
  const int64_t first = (int64_t)i * per * 64;
  *lo = first < vis ? (int)first : vis;
  const int64_t last = first + (int64_t)per * 64;
  *hi = last < vis ? (int)last : vis;
}

}  // namespace mi
