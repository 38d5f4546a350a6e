// RoPE of q and k at every sequence's own positions, and the append of k and v
// to a paged KV cache, in one launch.
//
// Math, for token s < n_b of row b at position p = start_b + s (rotate-half form,
// as in rope.hip):
//   y[i]       = x[i]       * cos[p, i] - x[i + D/2] * sin[p, i]
//   y[i + D/2] = x[i + D/2] * cos[p, i] + x[i]       * sin[p, i]
// in fp32, products and sum rounded separately.  The token's place is offset
// p % P of page table[b, p / P].  K pages are [kv head][P][D]; V pages are
// transposed, [kv head][D][P], which is the order in which the attention's
// matrix instructions take V (paged_attn_mfma.hpp).
//
// Pages of the activations' type take y rounded once and V's bits.  8-bit pages
// (e4m3) have one scale for each page, kv head and K / V, a power of two, so that
// taking an entry to another scale moves its exponent only (it loses bits only
// where it becomes subnormal) and a page that is filled token by token does not
// add up rounding errors:
//   need = the least 2^e >= max |new finite entries of the page| / 448, e >= -120
//   s    = need                 if the page's first entry is new
//        = max(s_old, need)     otherwise; older entries become e4m3(old * s_old / s)
//   entry = e4m3(x / s), rounded once from fp32; NaN for an infinity or NaN.
//
// One block per (row, page the row's tokens may touch, kv head); the blocks after
// those rotate q.  K moves 8 pairs a thread (16-byte loads), V blocks of 4 tokens x
// 8 dims a thread, packed in registers to 4 tokens of one dim (4 bytes in 8 bits,
// 8 bytes in 16): a row of the transposed page is written in whole 64- to 128-byte
// runs by neighbouring threads, without LDS.  8-bit pages read their tokens twice
// (largest value, then entries): the second read comes from the caches, and no
// register holds a page.  Other layouts (VEC = 1) move one element at a time.
//
// Long prompts are bound by memory, steps by the chain of dependent reads (row's position,
// page number, tokens, for 8-bit pages the largest value and the old scale).  Measured
// (kernel alone): 4 x 2048 tokens of 32 + 8 + 8 heads of 64, bf16 into 8-bit pages, 92.5 MB
// in 18.2 us, 5.1 TB/s; 1021 tokens of 128, fp16, 25.4 MB in 8.6 us; 64 rows of 4 tokens
// into 8-bit pages 8.0 us; one token 4.1 us, an empty launch being 2 to 3.
#include <initializer_list>

#include "common.hpp"
#include "paged_common.hpp"

namespace mi {

struct PagedAppendArgs {
  const void* xq;
  const void* xk;
  const void* xv;
  const void* cos;
  const void* sin;
  void* q_out;
  void* kp;
  void* vp;
  float* scales;
  const int32_t* table;
  const int64_t* start;   // null: start_pos for every row
  const int64_t* lens;    // null: S for every row
  int64_t start_pos;
  int64_t q_sb, q_sh, q_ss;
  int64_t k_sb, k_sh, k_ss;
  int64_t v_sb, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss;
  int64_t t_sb, c_ss, s_ss;
  int64_t table_rows, num_pages, q_items;
  int32_t H, Hkv, S, D, P, slots, spans, kv_blocks;
};

// Row b's first position and number of tokens; positions that no slot holds are cut off.
struct Span {
  int64_t start;    // position of token 0 (may be negative: those tokens have no place)
  int64_t first;    // first position with a place
  int64_t end;      // one past the last
};
__device__ inline Span row_span(const PagedAppendArgs& a, int b) {
  const int64_t cap = (int64_t)a.slots * a.P;
  int64_t st = a.start != nullptr ? a.start[b] : a.start_pos;
  int64_t n = a.lens != nullptr ? a.lens[b] : a.S;
  n = n < 0 ? 0 : (n > a.S ? a.S : n);
  st = st > cap ? cap : (st < -(int64_t)a.S ? -(int64_t)a.S : st);
  Span r;
  r.start = st;
  r.first = st > 0 ? st : 0;
  r.end = st + n < cap ? st + n : cap;
  return r;
}

__device__ inline int64_t table_row(const PagedAppendArgs& a, int64_t pos) {
  return pos < 0 ? 0 : (pos < a.table_rows ? pos : a.table_rows - 1);
}

// VEC consecutive elements to fp32
template <typename T, int VEC>
__device__ inline void load_f32(const T* p, float* o) {
  if constexpr (VEC == 8) {
    static_assert(sizeof(T) == 2, "16-byte groups are for 2-byte types");
    Chunk<T>::unpack(load16(p), o);
  } else {
    o[0] = Elem<T>::to_f32(p[0]);
  }
}
template <typename CT, int VEC>
__device__ inline void load_table(const CT* p, CT* o) {
  if constexpr (VEC == 8 && sizeof(CT) == 2) {
    typedef CT c8 __attribute__((ext_vector_type(8)));
    const c8 w = __builtin_bit_cast(c8, load16(p));
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = w[e];
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = p[e];
  }
}

// The rotation of VEC pairs; OT = T rounds to T, OT = float keeps fp32.
template <typename OT, typename CT, int VEC>
__device__ inline void rotate(const float* x1, const float* x2, const CT* c, const CT* s, OT* y1,
                              OT* y2) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) rope_rotate<OT, CT>(x1[e], x2[e], c[e], s[e], y1[e], y2[e]);
}

template <typename T, int VEC>
__device__ inline void store_t(T* p, const T* y) {
  if constexpr (VEC == 8) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    t8 w;
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = y[e];
    *reinterpret_cast<u32x4*>(p) = __builtin_bit_cast(u32x4, w);
  } else {
    p[0] = y[0];
  }
}

__device__ inline float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.0f;   // an infinity or NaN has no say in the scale
}

// the rotated pairs (i0.., i0 + D/2..) of token s, in fp32
template <typename T, typename CT, int VEC>
__device__ inline void rotated_k(const PagedAppendArgs& a, const T* row, int64_t pos, int i0,
                                 float* y1, float* y2) {
  const int half = a.D >> 1;
  float x1[VEC], x2[VEC];
  CT c[VEC], s[VEC];
  const int64_t cr = table_row(a, pos);
  load_f32<T, VEC>(row + i0, x1);
  load_f32<T, VEC>(row + half + i0, x2);
  load_table<CT, VEC>(reinterpret_cast<const CT*>(a.cos) + cr * a.c_ss + i0, c);
  load_table<CT, VEC>(reinterpret_cast<const CT*>(a.sin) + cr * a.s_ss + i0, s);
  rotate<float, CT, VEC>(x1, x2, c, s, y1, y2);
}

// Largest value of the block (at most 4 waves), in every thread.
__device__ inline float block_max(float x, float* lds) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m, 64));
  __syncthreads();   // lds may hold the last call's values
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  x = lds[0];
  for (int w = 1; w < (int)(blockDim.x >> 6); ++w) x = fmaxf(x, lds[w]);
  return x;
}

template <typename T, typename CT, int VEC, bool E8>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a) {
  const int half = a.D >> 1, tid = threadIdx.x, nt = blockDim.x;
  const int per_tok = half / VEC;     // K items of a token
  if ((int64_t)blockIdx.x >= a.kv_blocks) {   // q: a thread rotates VEC pairs
    const int64_t step = (int64_t)(gridDim.x - a.kv_blocks) * nt;
    for (int64_t it = (int64_t)(blockIdx.x - a.kv_blocks) * nt + tid; it < a.q_items; it += step) {
      int64_t r = it;
      const int i0 = (int)(r % per_tok) * VEC; r /= per_tok;
      const int h = (int)(r % a.H); r /= a.H;
      const int s = (int)(r % a.S);
      const int b = (int)(r / a.S);
      const T* xp = reinterpret_cast<const T*>(a.xq) + b * a.q_sb + h * a.q_sh + s * a.q_ss;
      T* op = reinterpret_cast<T*>(a.q_out) + b * a.o_sb + h * a.o_sh + s * a.o_ss;
      const int64_t st = a.start != nullptr ? a.start[b] : a.start_pos;
      // (a position past either end of the table takes its nearest row; no sum overflows)
      const int64_t cr = table_row(a, st > a.table_rows ? a.table_rows
                                      : (st < -(int64_t)a.S ? 0 : st + s));
      float x1[VEC], x2[VEC];
      CT c[VEC], sn[VEC];
      T y1[VEC], y2[VEC];
      load_f32<T, VEC>(xp + i0, x1);
      load_f32<T, VEC>(xp + half + i0, x2);
      load_table<CT, VEC>(reinterpret_cast<const CT*>(a.cos) + cr * a.c_ss + i0, c);
      load_table<CT, VEC>(reinterpret_cast<const CT*>(a.sin) + cr * a.s_ss + i0, sn);
      rotate<T, CT, VEC>(x1, x2, c, sn, y1, y2);
      store_t<T, VEC>(op + i0, y1);
      store_t<T, VEC>(op + half + i0, y2);
    }
    return;
  }

  // one (row b, touched page `span`, kv head h)
  int blk = blockIdx.x;
  const int h = blk % a.Hkv; blk /= a.Hkv;
  const int span = blk % a.spans;
  const int b = blk / a.spans;
  const Span r = row_span(a, b);
  const int64_t slot = r.first / a.P + span;
  const int64_t page0 = slot * a.P;                       // the page's first position
  const int64_t lo = r.first > page0 ? r.first : page0;   // new positions [lo, hi)
  const int64_t hi = r.end < page0 + a.P ? r.end : page0 + a.P;
  if (lo >= hi) return;                                   // (also slot >= slots: hi <= end <= cap)
  const int32_t page = a.table[(int64_t)b * a.t_sb + slot];
  if (page < 0 || page >= a.num_pages) return;            // no such page: no place
  const int off = (int)(lo - page0), n = (int)(hi - lo), s0 = (int)(lo - r.start);
  const int64_t ph = (int64_t)page * a.Hkv + h;
  const T* xk = reinterpret_cast<const T*>(a.xk) + b * a.k_sb + h * a.k_sh + s0 * a.k_ss;
  const T* xv = reinterpret_cast<const T*>(a.xv) + b * a.v_sb + h * a.v_sh + s0 * a.v_ss;
  const int64_t tile = ph * a.P * a.D;
  // V items: 4 tokens of the page (aligned to 4 offsets) x VEC dims
  const int vdims = a.D / VEC, q0 = off >> 2, quads = ((off + n + 3) >> 2) - q0;

  float kinv = 1.0f, vinv = 1.0f;
  if constexpr (E8) {
    __shared__ float red[4];
    float km = 0.0f, vm = 0.0f;
    for (int it = tid; it < n * per_tok; it += nt) {
      const int t = it / per_tok, i0 = (it % per_tok) * VEC;
      float y1[VEC], y2[VEC];
      rotated_k<T, CT, VEC>(a, xk + t * a.k_ss, lo + t, i0, y1, y2);
#pragma unroll
      for (int e = 0; e < VEC; ++e) km = fmaxf(km, fmaxf(finite_abs(y1[e]), finite_abs(y2[e])));
    }
    for (int it = tid; it < n * vdims; it += nt) {
      float x[VEC];
      load_f32<T, VEC>(xv + (it / vdims) * a.v_ss + (it % vdims) * VEC, x);
#pragma unroll
      for (int e = 0; e < VEC; ++e) vm = fmaxf(vm, finite_abs(x[e]));
    }
    km = block_max(km, red);
    vm = block_max(vm, red);
    float ks = e4m3_scale(km), vs = e4m3_scale(vm);
    float* sc = a.scales + 2 * ph;
    if (off > 0) {
      const float k_old = sc[0], v_old = sc[1];
      ks = fmaxf(ks, k_old);
      vs = fmaxf(vs, v_old);
      uint8_t* kt = reinterpret_cast<uint8_t*>(a.kp) + tile;
      uint8_t* vt = reinterpret_cast<uint8_t*>(a.vp) + tile;
      // (bytes: a dword may hold entries that other threads write below)
      if (ks != k_old)
        for (int i = tid; i < off * a.D; i += nt)
          kt[i] = to_e4m3(from_e4m3(kt[i]) * (k_old / ks));
      if (vs != v_old)
        for (int i = tid; i < off * a.D; i += nt) {
          uint8_t* p = vt + (int64_t)(i / off) * a.P + i % off;
          *p = to_e4m3(from_e4m3(*p) * (v_old / vs));
        }
    }
    __syncthreads();   // every thread has read the old scales
    if (tid == 0) {
      sc[0] = ks;
      sc[1] = vs;
    }
    kinv = 1.0f / ks;  // exact: powers of two between 2^-120 and 2^120
    vinv = 1.0f / vs;
  }

  for (int it = tid; it < n * per_tok; it += nt) {
    const int t = it / per_tok, i0 = (it % per_tok) * VEC;
    float y1[VEC], y2[VEC];
    rotated_k<T, CT, VEC>(a, xk + t * a.k_ss, lo + t, i0, y1, y2);
    const int64_t at = tile + (int64_t)(off + t) * a.D + i0;
    if constexpr (E8) {
      uint8_t* p = reinterpret_cast<uint8_t*>(a.kp) + at;
      if constexpr (VEC == 8) {
        *reinterpret_cast<uint64_t*>(p) = pack8_e4m3(y1, kinv);
        *reinterpret_cast<uint64_t*>(p + half) = pack8_e4m3(y2, kinv);
      } else {
        p[0] = to_e4m3(y1[0] * kinv);
        p[half] = to_e4m3(y2[0] * kinv);
      }
    } else {
      T* p = reinterpret_cast<T*>(a.kp) + at;
      T t1[VEC], t2[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        t1[e] = Elem<T>::from_f32(y1[e]);
        t2[e] = Elem<T>::from_f32(y2[e]);
      }
      store_t<T, VEC>(p, t1);
      store_t<T, VEC>(p + half, t2);
    }
  }

  for (int it = tid; it < quads * vdims; it += nt) {
    // neighbouring threads take neighbouring quads of the same dims
    const int qd = q0 + it % quads, d0 = (it / quads) * VEC;
    const int t0 = 4 * qd - off;              // token of the quad's first offset (may be < 0)
    const bool whole = t0 >= 0 && t0 + 4 <= n;
    if constexpr (E8) {
      float x[4][VEC];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (t0 + j >= 0 && t0 + j < n) {
          load_f32<T, VEC>(xv + (t0 + j) * a.v_ss + d0, x[j]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[j][e] = 0.0f;
        }
      }
      uint8_t* p = reinterpret_cast<uint8_t*>(a.vp) + tile + (int64_t)d0 * a.P + 4 * qd;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t w = pack4_e4m3(x[0][e] * vinv, x[1][e] * vinv, x[2][e] * vinv, x[3][e] * vinv);
        if (whole) {
          *reinterpret_cast<uint32_t*>(p + (int64_t)e * a.P) = w;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (t0 + j >= 0 && t0 + j < n) p[(int64_t)e * a.P + j] = (uint8_t)(w >> (8 * j));
        }
      }
    } else {
      T x[4][VEC];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (t0 + j >= 0 && t0 + j < n) {
          load_table<T, VEC>(xv + (t0 + j) * a.v_ss + d0, x[j]);
        } else {
#pragma unroll
          for (int e = 0; e < VEC; ++e) x[j][e] = (T)0.0f;
        }
      }
      T* p = reinterpret_cast<T*>(a.vp) + tile + (int64_t)d0 * a.P + 4 * qd;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (whole) {
          typedef T t4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<t4*>(p + (int64_t)e * a.P) = t4{x[0][e], x[1][e], x[2][e], x[3][e]};
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (t0 + j >= 0 && t0 + j < n) p[(int64_t)e * a.P + j] = x[j][e];
        }
      }
    }
  }
}

namespace {

template <typename T, typename CT>
void launch_append(const PagedAppendArgs& a, int grid, int block, bool vec, bool e8,
                   hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (vec) {
      if (e8)
        hipLaunchKernelGGL((paged_append_kernel<T, CT, 8, true>), dim3(grid), dim3(block), 0, st, a);
      else
        hipLaunchKernelGGL((paged_append_kernel<T, CT, 8, false>), dim3(grid), dim3(block), 0, st, a);
      return;
    }
  }
  if (e8)
    hipLaunchKernelGGL((paged_append_kernel<T, CT, 1, true>), dim3(grid), dim3(block), 0, st, a);
  else
    hipLaunchKernelGGL((paged_append_kernel<T, CT, 1, false>), dim3(grid), dim3(block), 0, st, a);
}

bool aligned16(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if ((uintptr_t)p % 16 != 0) return false;
  return true;
}
bool rows16(int64_t es, std::initializer_list<int64_t> strides) {
  for (int64_t s : strides)
    if ((s * es) % 16 != 0) return false;
  return true;
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int32_t mi_rope_paged_append(
    const void* xq, const void* xk, const void* xv, const void* cos, const void* sin,
    void* q_out, void* k_pages, void* v_pages, float* scales, const int32_t* page_table,
    int64_t start_pos, const int64_t* start, const int64_t* query_lens, int64_t table_rows,
    int64_t batch, int64_t n_heads, int64_t n_kv_heads, int64_t seq_len, int64_t head_dim,
    int64_t num_pages, int64_t page_size, int64_t slots, int64_t xq_sb, int64_t xq_sh,
    int64_t xq_ss, int64_t xk_sb, int64_t xk_sh, int64_t xk_ss, int64_t xv_sb, int64_t xv_sh,
    int64_t xv_ss, int64_t qo_sb, int64_t qo_sh, int64_t qo_ss, int64_t pt_sb, int64_t c_ss,
    int64_t s_ss, int32_t dtype, int32_t cdtype, int32_t store, void* stream) {
  if (xk == nullptr || xv == nullptr || cos == nullptr || sin == nullptr || k_pages == nullptr ||
      v_pages == nullptr || page_table == nullptr || ((xq == nullptr) != (q_out == nullptr))) {
    set_last_error("rope_paged_append: null pointer");
    return MI_ERR_INVALID;
  }
  if (int32_t st = paged_check("rope_paged_append", batch, n_heads, n_kv_heads, seq_len, head_dim,
                               num_pages, page_size, slots, dtype, store, scales))
    return st;
  if (head_dim % 2 != 0) {
    set_last_error("rope_paged_append: head_dim must be even, got %lld", (long long)head_dim);
    return MI_ERR_INVALID;
  }
  if (table_rows < 1) {
    set_last_error("rope_paged_append: cos/sin have no rows");
    return MI_ERR_INVALID;
  }
  if (cdtype != dtype && cdtype != MI_DTYPE_F32) {
    set_last_error("rope_paged_append: cos/sin must have the activations' dtype or fp32");
    return MI_ERR_INVALID;
  }
  if (batch == 0 || seq_len == 0) return MI_OK;
  PagedAppendArgs a{};
  a.xq = xq; a.xk = xk; a.xv = xv; a.cos = cos; a.sin = sin;
  a.q_out = q_out; a.kp = k_pages; a.vp = v_pages; a.scales = scales;
  a.table = page_table; a.start = start; a.lens = query_lens; a.start_pos = start_pos;
  a.q_sb = xq_sb; a.q_sh = xq_sh; a.q_ss = xq_ss;
  a.k_sb = xk_sb; a.k_sh = xk_sh; a.k_ss = xk_ss;
  a.v_sb = xv_sb; a.v_sh = xv_sh; a.v_ss = xv_ss;
  a.o_sb = qo_sb; a.o_sh = qo_sh; a.o_ss = qo_ss;
  a.t_sb = pt_sb; a.c_ss = c_ss; a.s_ss = s_ss;
  a.table_rows = table_rows; a.num_pages = num_pages;
  a.H = (int32_t)n_heads; a.Hkv = (int32_t)n_kv_heads; a.S = (int32_t)seq_len;
  a.D = (int32_t)head_dim; a.P = (int32_t)page_size; a.slots = (int32_t)slots;
  const int es = dtype == MI_DTYPE_F32 ? 4 : 2;
  const bool vec = es == 2 && head_dim % 16 == 0 &&
                   aligned16({xk, xv, cos, sin, k_pages, v_pages}) &&
                   (xq == nullptr || (aligned16({xq, q_out}) &&
                                      rows16(2, {xq_sb, xq_sh, xq_ss, qo_sb, qo_sh, qo_ss}))) &&
                   rows16(2, {xk_sb, xk_sh, xk_ss, xv_sb, xv_sh, xv_ss}) &&
                   rows16(cdtype == MI_DTYPE_F32 ? 4 : 2, {c_ss, s_ss});
  // pages that seq_len tokens touch at most, wherever the first of them lies
  a.spans = (int32_t)((seq_len + page_size - 2) / page_size + 1);
  const int64_t kv_blocks = batch * a.spans * n_kv_heads;
  // 4 waves for a page of a prompt; one wave where a block has a few tokens (4 x 2048 tokens
  // 21.4 us, with one wave 25.5; 64 rows of 4 tokens 10.3 us, with 4 waves 12.1)
  const int block = seq_len > 8 ? 256 : 64;
  a.q_items = xq == nullptr ? 0 : batch * seq_len * n_heads * (head_dim / 2 / (vec ? 8 : 1));
  int64_t q_blocks = (a.q_items + block - 1) / block;
  if (q_blocks > 16384) q_blocks = 16384;   // the kernel loops over the rest
  if (kv_blocks + q_blocks > INT32_MAX) {
    set_last_error("rope_paged_append: too many rows and pages for one call");
    return MI_ERR_UNSUPPORTED;
  }
  a.kv_blocks = (int32_t)kv_blocks;
  const int grid = (int)(kv_blocks + q_blocks);
  const bool e8 = store == MI_STORE_E4M3;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MI_DTYPE_F32)
    launch_append<float, float>(a, grid, block, vec, e8, st);
  else if (dtype == MI_DTYPE_BF16 && cdtype == MI_DTYPE_F32)
    launch_append<bf16_t, float>(a, grid, block, vec, e8, st);
  else if (dtype == MI_DTYPE_BF16)
    launch_append<bf16_t, bf16_t>(a, grid, block, vec, e8, st);
  else if (cdtype == MI_DTYPE_F32)
    launch_append<f16_t, float>(a, grid, block, vec, e8, st);
  else
    launch_append<f16_t, f16_t>(a, grid, block, vec, e8, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_last_error("rope_paged_append: launch failed: %s", hipGetErrorString(e));
    return (int32_t)e;
  }
  return MI_OK;
}
