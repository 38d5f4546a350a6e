// Attention of the newest tokens over a paged KV cache: host side, the kernel for the
// head_dims that are not 64, 128 or 256, and its join of split keys.
//
// out[b, h, s] = sum_j softmax_j(scale * q[b, h, s] . k[j]) v[j] over the keys
// j < seq_lens[b] - n_b + s + 1 of row b (n_b query tokens, the newest of its
// keys); 0 for a row that sees none.
//
// head_dim 64, 128 and 256 run on the matrix cores (paged_attn_mfma.hpp).  For the others
// up to 256 paged_attn_kernel (below) computes it in fp32, one block for each (row, head,
// token, key range), a wave taking 64 keys at a time: the lane's key against q from LDS,
// the softmax across the wave, then a lane per dim over the transposed V.  Bound by its
// scalar products: a block has one query row, so each of the group's rows reads the keys
// again (8 rows of 2048 fp32 keys, 32 heads over 8 of 128, took 62.7 us on it and take
// 33.9 on the matrix cores).
#include <initializer_list>

#include "paged_attn_kernels.hpp"

namespace mi {

// One entry of a page in fp32 (the scale is applied to sums, not to entries).
template <typename T, bool E8>
struct Entry {
  typedef T type;
  static __device__ inline float get(const T* p) { return Elem<T>::to_f32(*p); }
};
template <typename T>
struct Entry<T, true> {
  typedef uint8_t type;
  static __device__ inline float get(const uint8_t* p) { return from_e4m3(*p); }
};

// N entries from p, aligned to N * sizeof(entry) or 16 bytes
template <typename T, bool E8, int N>
__device__ inline void entries(const typename Entry<T, E8>::type* p, float* o) {
  if constexpr (E8) {
    static_assert(N == 16, "16 entries are one 16-byte load");
    const u32x4 w = load16(p);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[4 * i] = __builtin_amdgcn_cvt_f32_fp8((int)u[i], 0);
      o[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8((int)u[i], 1);
      o[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8((int)u[i], 2);
      o[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8((int)u[i], 3);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; i += Chunk<T>::kN) Chunk<T>::unpack(load16(p + i), o + i);
  }
}

template <typename T, bool E8>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedAttnArgs a) {
  typedef Entry<T, E8> En;
  typedef typename En::type E;
  __shared__ float qs[256];
  __shared__ float acc_s[4][256];
  __shared__ float ml_s[4][2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t blk = blockIdx.x;
  const int split = (int)(blk % a.splits); blk /= a.splits;
  const int64_t row = blk;                       // (b * Hq + h) * S + s
  const int s = (int)(row % a.S);
  const int h = (int)(row / a.S % a.Hq), b = (int)(row / a.S / a.Hq);
  const RowKeys rk = row_keys(a, b);
  int lo, hi;
  split_range(rk.vis(s), split, a.splits, &lo, &hi);

  const T* qp = reinterpret_cast<const T*>(a.q) + b * a.q_sb + h * a.q_sh + s * a.q_ss;
  for (int d = tid; d < a.D; d += 256) qs[d] = Elem<T>::to_f32(qp[d]);
  __syncthreads();

  const int hk = h / a.group;
  const int64_t page_elems = (int64_t)a.P * a.D;
  const E* kp = reinterpret_cast<const E*>(a.kp) + hk * page_elems;
  const E* vp = reinterpret_cast<const E*>(a.vp) + hk * page_elems;
  const int32_t* table = a.table + (int64_t)b * a.t_sb;
  const bool wide = a.D % 16 == 0;               // K rows are whole 16-byte chunks
  float m = kLowest, l = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};

  for (int k0 = lo + 64 * wave; k0 < hi; k0 += 256) {
    const int key = k0 + lane;
    const int32_t page = key < hi ? table[key >> a.p_shift] : -1;
    const bool live = page >= 0 && page < a.num_pages;
    float x = -INFINITY, vs = 1.0f;
    if (live) {
      const E* kr = kp + (int64_t)page * a.Hkv * page_elems + (int64_t)(key & (a.P - 1)) * a.D;
      float dot = 0.0f;
      if (wide) {
        for (int d = 0; d < a.D; d += 16) {
          float kv[16];
          entries<T, E8, 16>(kr + d, kv);
#pragma unroll
          for (int e = 0; e < 16; ++e) dot = fmaf(qs[d + e], kv[e], dot);
        }
      } else {
        for (int d = 0; d < a.D; ++d) dot = fmaf(qs[d], En::get(kr + d), dot);
      }
      if constexpr (E8) {
        const float* sc = a.scales + 2 * ((int64_t)page * a.Hkv + hk);
        dot *= sc[0];
        vs = sc[1];
      }
      x = dot * a.scale_log2;
    }
    float top = x;
#pragma unroll
    for (int i = 32; i; i >>= 1) top = fmaxf(top, __shfl_xor(top, i, 64));
    const float m_new = fmaxf(m, top);
    const float alpha = fast_exp2(m - m_new);
    const float p = live ? fast_exp2(x - m_new) : 0.0f;
    float sum = p;
#pragma unroll
    for (int i = 32; i; i >>= 1) sum += __shfl_xor(sum, i, 64);
    l = l * alpha + sum;
    m = m_new;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= alpha;
    const float pv = p * vs;   // the V scale belongs to the key's page
    for (int c = 0; c < 4; ++c) {                // 16 keys lie in one page
      const int kc = k0 + 16 * c;
      if (kc >= hi) break;
      const int32_t pg = __shfl(page, 16 * c, 64);
      if (pg < 0 || pg >= a.num_pages) continue;
      const int n = hi - kc < 16 ? hi - kc : 16;
      const E* vr = vp + (int64_t)pg * a.Hkv * page_elems + (kc & (a.P - 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (64 * i >= a.D) break;
        float v[16];
        if (d < a.D) {
          entries<T, E8, 16>(vr + (int64_t)d * a.P, v);
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float pj = __shfl(pv, 16 * c + j, 64);
          if (j < n) acc[i] = fmaf(pj, v[j], acc[i]);   // keys behind the last are not added
        }
      }
    }
  }

  // the block's waves
#pragma unroll
  for (int i = 0; i < 4; ++i) acc_s[wave][lane + 64 * i] = acc[i];
  if (lane == 0) {
    ml_s[wave][0] = m;
    ml_s[wave][1] = l;
  }
  __syncthreads();
  float M = kLowest, L = 0.0f, w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) M = fmaxf(M, ml_s[i][0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = fast_exp2(ml_s[i][0] - M);
    L += w[i] * ml_s[i][1];
  }
  if (tid < a.D) {
    float o = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) o += w[i] * acc_s[i][tid];
    if (a.splits == 1) {
      T* op = reinterpret_cast<T*>(a.out) + b * a.o_sb + h * a.o_sh + s * a.o_ss;
      op[tid] = Elem<T>::from_f32(L == 0.0f ? 0.0f : o / L);
    } else {
      a.part_acc[(row * a.splits + split) * a.D + tid] = o;
    }
  }
  if (tid == 0) {
    if (a.splits > 1) {
      a.part_ml[2 * (row * a.splits + split)] = M;
      a.part_ml[2 * (row * a.splits + split) + 1] = L;
    } else if (a.lse != nullptr) {
      a.lse[row] = L == 0.0f ? -INFINITY : (M + fast_log2(L)) * kLn2;
    }
  }
}

// The splits of a row joined: sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i.  A block
// takes a row and its waves every 4th split, a lane dims lane, lane + 64, .., four splits'
// loads in flight.
template <typename T>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
  __shared__ float acc_s[4][256];
  __shared__ float l_s[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const float* ml = a.part_ml + 2 * row * a.splits;
  const float* pa = a.part_acc + row * a.splits * a.D;
  float M = kLowest;
  for (int i = lane; i < a.splits; i += 64) M = fmaxf(M, ml[2 * i]);
#pragma unroll
  for (int i = 32; i; i >>= 1) M = fmaxf(M, __shfl_xor(M, i, 64));
  float L = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = wave; i < a.splits; i += 16) {
    float l[4], w[4], x[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = i + 4 * j < a.splits;
      const int s = in ? i + 4 * j : i;
      l[j] = in ? ml[2 * s + 1] : 0.0f;
      w[j] = ml[2 * s];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[j][k] = lane + 64 * k < a.D ? pa[(int64_t)s * a.D + lane + 64 * k] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (l[j] == 0.0f) continue;                // an empty range has no sums
      const float f = fast_exp2(w[j] - M);
      L += f * l[j];
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += f * x[j][k];
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) acc_s[wave][lane + 64 * k] = o[k];
  if (lane == 0) l_s[wave] = L;
  __syncthreads();
  L = (l_s[0] + l_s[1]) + (l_s[2] + l_s[3]);
  const int s = (int)(row % a.S);
  const int h = (int)(row / a.S % a.Hq), b = (int)(row / a.S / a.Hq);
  T* op = reinterpret_cast<T*>(a.out) + b * a.o_sb + h * a.o_sh + s * a.o_ss;
  if (tid < a.D) {
    const float y = (acc_s[0][tid] + acc_s[1][tid]) + (acc_s[2][tid] + acc_s[3][tid]);
    op[tid] = Elem<T>::from_f32(L == 0.0f ? 0.0f : y / L);
  }
  if (tid == 0 && a.lse != nullptr)
    a.lse[row] = L == 0.0f ? -INFINITY : (M + fast_log2(L)) * kLn2;
}

namespace {

template <typename T>
int32_t launch_attn(const PagedAttnArgs& a, bool e8, hipStream_t st) {
  const int64_t rows = (int64_t)a.B * a.Hq * a.S, blocks = rows * a.splits;
  if (blocks > INT32_MAX) {
    set_last_error("paged_attn: too many rows and splits for one call");
    return MI_ERR_UNSUPPORTED;
  }
  if (e8)
    hipLaunchKernelGGL((paged_attn_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_attn_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  if (a.splits > 1)
    hipLaunchKernelGGL(paged_join_kernel<T>, dim3((unsigned)rows), dim3(256), 0, st, a);
  return MI_OK;
}

}  // namespace
}  // namespace mi

using namespace mi;

// num_splits counts parts of a KV head's keys over all rows; paged_attn_kernel divides each
// row's keys alike.
static int64_t ranges_per_row(int64_t num_splits, int64_t batch) {
  const int64_t n = num_splits / batch;
  return n < 1 ? 1 : (n > 256 ? 256 : n);
}

extern "C" int64_t mi_paged_attn_splits(int64_t batch, int64_t n_heads, int64_t n_kv_heads,
                                        int64_t seq_len, int64_t head_dim, int64_t page_size,
                                        int64_t slots, int32_t dtype, int32_t store) {
  if (batch <= 0 || n_heads <= 0 || n_kv_heads <= 0 || seq_len <= 0 || slots <= 0 ||
      page_size <= 0 || slots > INT32_MAX / page_size || batch > (1 << 24) ||
      n_heads > (1 << 16) || n_heads % n_kv_heads != 0 || seq_len > (1 << 24))
    return 1;
  const int64_t units = (slots * page_size + 63) / 64;
  const PagedPlan plan = paged_plan(batch, n_heads, n_kv_heads, seq_len, head_dim, dtype, 1);
  if (plan.mfma) {
    const int64_t entry = store == MI_STORE_E4M3 ? 1 : dtype == MI_DTYPE_F32 ? 4 : 2;
    return paged_mfma_splits(plan, batch, n_kv_heads, head_dim, units, entry);
  }
  const int64_t blocks = batch * n_heads * seq_len;
  // 8 blocks of 4 waves a compute unit, of 4 units of 64 keys or more each; a multiple of the
  // 8 L2s, so that the heads of a group, which read the same keys, find them in one (1 row of
  // up to 32768 fp16 keys, 24 heads over 8 of 96: 64 splits 62 us, 85 132, 128 65; 16 rows of up
  // to 8192, 32 over 8 of 80: 4 splits 104 us, 8 96, 16 105)
  int64_t s = (8 * (int64_t)device_cu_count() / blocks + 7) / 8 * 8;
  if (s > (units + 3) / 4) s = (units + 3) / 4;
  if (s > 8) s = s / 8 * 8;
  return ranges_per_row(s * batch, batch) * batch;
}

extern "C" int64_t mi_paged_attn_workspace(int64_t batch, int64_t n_heads, int64_t n_kv_heads,
                                           int64_t seq_len, int64_t head_dim, int64_t num_splits,
                                           int32_t dtype) {
  if (batch <= 0 || n_heads <= 0 || n_kv_heads <= 0 || seq_len <= 0 || head_dim <= 0 ||
      num_splits <= 1 || num_splits > MI_PAGED_ATTN_MAX_SPLITS || batch > (1 << 24) ||
      n_heads > (1 << 16) || n_heads % n_kv_heads != 0 || seq_len > (1 << 24) || head_dim > 256)
    return 0;
  const PagedPlan plan =
      paged_plan(batch, n_heads, n_kv_heads, seq_len, head_dim, dtype, num_splits);
  if (plan.mfma) return paged_mfma_workspace(plan, n_kv_heads, head_dim);
  const int64_t n = ranges_per_row(num_splits, batch);
  return n > 1 ? batch * n_heads * seq_len * n * (head_dim + 2) : 0;
}

extern "C" int32_t mi_paged_attn(
    const void* q, const void* k_pages, const void* v_pages, const float* scales,
    const int32_t* page_table, const int64_t* seq_lens, const int64_t* query_lens, float* part,
    int64_t part_elems, void* out, float* lse, int64_t batch, int64_t n_heads,
    int64_t n_kv_heads, int64_t seq_len, int64_t head_dim, int64_t num_pages, int64_t page_size,
    int64_t slots, int64_t num_splits, int64_t q_sb, int64_t q_sh, int64_t q_ss, int64_t o_sb,
    int64_t o_sh, int64_t o_ss, int64_t pt_sb, float sm_scale, int32_t dtype, int32_t store,
    void* stream) {
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || page_table == nullptr ||
      seq_lens == nullptr || out == nullptr) {
    set_last_error("paged_attn: null pointer");
    return MI_ERR_INVALID;
  }
  if (int32_t st = paged_check("paged_attn", batch, n_heads, n_kv_heads, seq_len, head_dim,
                               num_pages, page_size, slots, dtype, store, scales))
    return st;
  if (num_splits < 1 || num_splits > MI_PAGED_ATTN_MAX_SPLITS) {
    set_last_error("paged_attn: num_splits must be 1..%d, got %lld", MI_PAGED_ATTN_MAX_SPLITS,
                   (long long)num_splits);
    return MI_ERR_INVALID;
  }
  if (!(sm_scale > 0.0f) || sm_scale > 3.402823466e38f) {
    set_last_error("paged_attn: sm_scale must be positive and finite");
    return MI_ERR_INVALID;
  }
  if ((uintptr_t)k_pages % 16 != 0 || (uintptr_t)v_pages % 16 != 0) {
    set_last_error("paged_attn: pages must be 16-byte aligned");
    return MI_ERR_INVALID;
  }
  if (batch == 0 || seq_len == 0) return MI_OK;
  const int64_t rows = batch * n_heads * seq_len;
  const PagedPlan plan =
      paged_plan(batch, n_heads, n_kv_heads, seq_len, head_dim, dtype, num_splits);
  const int64_t ranges = plan.mfma ? 1 : ranges_per_row(num_splits, batch);
  // (units of a list, blocks and rows are 32-bit)
  if (rows > INT32_MAX || rows * ranges > INT32_MAX || plan.tiles > 65535 ||
      n_kv_heads * (plan.parts > batch ? plan.parts : batch) > INT32_MAX ||
      n_kv_heads * batch * plan.tiles > INT32_MAX ||
      batch * ((slots * page_size + 63) / 64) > INT32_MAX ||
      n_kv_heads * page_size * head_dim * 4 > UINT32_MAX) {
    set_last_error("paged_attn: too many rows, keys and splits for one call");
    return MI_ERR_UNSUPPORTED;
  }
  const int64_t need =
      mi_paged_attn_workspace(batch, n_heads, n_kv_heads, seq_len, head_dim, num_splits, dtype);
  if (need > 0 && (part == nullptr || (uintptr_t)part % 16 != 0 || part_elems < need)) {
    set_last_error("paged_attn: %lld splits need a 16-byte aligned workspace of %lld floats",
                   (long long)num_splits, (long long)need);
    return MI_ERR_INVALID;
  }
  PagedAttnArgs a{};
  a.q = q; a.kp = k_pages; a.vp = v_pages; a.scales = scales; a.table = page_table;
  a.seq_lens = seq_lens; a.lens = query_lens;
  a.part_acc = part;
  a.part_ml = need > 0 ? part + need / (head_dim + 2) * head_dim : nullptr;
  a.out = out; a.lse = lse;
  a.q_sb = q_sb; a.q_sh = q_sh; a.q_ss = q_ss;
  a.o_sb = o_sb; a.o_sh = o_sh; a.o_ss = o_ss;
  a.t_sb = pt_sb; a.num_pages = num_pages;
  a.B = (int32_t)batch; a.Hq = (int32_t)n_heads; a.Hkv = (int32_t)n_kv_heads;
  a.group = (int32_t)(n_heads / n_kv_heads); a.S = (int32_t)seq_len; a.D = (int32_t)head_dim;
  a.P = (int32_t)page_size; a.p_shift = __builtin_ctzll((unsigned long long)page_size);
  a.slots = (int32_t)slots; a.splits = (int32_t)ranges;
  a.tiles = (int32_t)plan.tiles; a.parts = (int32_t)plan.parts; a.kv_rows = 16 * plan.r;
  a.scale_log2 = sm_scale * kLog2e;
  const bool e8 = store == MI_STORE_E4M3;
  const int64_t es = dtype == MI_DTYPE_F32 ? 4 : 2;
  auto rows_of = [&](const void* p, int64_t n, std::initializer_list<int64_t> strides) {
    bool ok = (uintptr_t)p % n == 0;
    for (int64_t s : strides) ok = ok && (s * es) % n == 0;
    return ok;
  };
  a.q_vec = rows_of(q, 16, {q_sb, q_sh, q_ss});
  a.o_vec = rows_of(out, 4 * es, {o_sb, o_sh, o_ss});
  hipStream_t st = (hipStream_t)stream;
  int32_t rc = MI_OK;
  if (plan.mfma)
    paged_attn_mfma_launch(a, plan, dtype, e8, st);
  else if (dtype == MI_DTYPE_BF16)
    rc = launch_attn<bf16_t>(a, e8, st);
  else if (dtype == MI_DTYPE_F16)
    rc = launch_attn<f16_t>(a, e8, st);
  else
    rc = launch_attn<float>(a, e8, st);
  if (rc != MI_OK) return rc;
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_last_error("paged_attn: launch failed: %s", hipGetErrorString(e));
    return (int32_t)e;
  }
  return MI_OK;
}
