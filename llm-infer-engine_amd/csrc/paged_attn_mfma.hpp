// Attention over a paged KV cache on the matrix cores: bf16 / fp16 queries, pages of
// the same type or of 8-bit floats, head_dims that are multiples of 64.
//
// A wave holds R tiles of 16 query rows of one KV head (row = token * group + head of
// the group) and streams its keys from memory straight into matrix operands: nothing
// passes through LDS until the end.  Per step of 64 keys (8-bit pages) or 32:
//   S^T = K Q^T      v_mfma_f32_16x16x32: A = 16 keys x 32 dims, B = 32 dims x 16 rows.
//                    A lane's operand is 8 dims of one key; the order of the dims is
//                    free as long as Q has the same, so each lane takes whole 16-byte
//                    pieces of its key.
//   softmax          the accumulator gives lane (g, r) = (lane / 16, lane % 16) four
//                    keys of row r per tile.  Which key is which row of A is free too:
//                    tile t's row 4g + i is key g * CK + 4t + i (CK = 16 or 8), so
//                    that lane (g, r) ends up with the CK neighbouring keys g * CK ..
//                    of row r, and the row's largest score is two lane swaps away.
//   O^T += V^T P^T   A = 16 dims x 32 keys, B = 32 keys x 16 rows.  P^T's lane (g, r)
//                    needs 8 keys of row r: those it already has (no shuffle), and
//                    V^T's lane the same 8 keys of one dim: 8 or 16 neighbouring entries
//                    of the transposed V page, one 16-byte load.
// 8-bit entries become bf16 (K: q's type) two at a time with v_cvt_scalef32_pk, exactly;
// V's page scale is the instruction's scale operand (bf16 has fp32's range, so no page
// overflows), K's multiplies the scores.  p goes in as a 16-bit value and its remainder
// (two products): off by 2^-16 at most, where one rounding of p to q's type would add an
// error as large as that of the output itself.  l sums p in fp32.
//
// KEYS: the block's 4 waves take every 4th step of the block's key range and join
// through LDS at the end (few rows: one token, a few drafts).  ROWS: the waves take
// different row tiles over the same keys, which then come from the caches (a piece of
// a prompt).  With PIPE two register sets alternate: the next step's 16 KB a wave are
// on their way while this one is multiplied; page numbers are fetched a step earlier.
//
// Keys behind the last visible one: their scores are -inf and their V entries are
// zeroed, so that nothing in them (a NaN in an old page) reaches a sum.  Where
// several tokens see different numbers of keys and one of those keys has a V entry that
// is not finite, the products take it as 0 and it is added to the rows that see it.
#pragma once

#include <type_traits>

#include "paged_attn_kernels.hpp"

namespace mi {

template <typename T> struct MatOp;
template <> struct MatOp<bf16_t> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static __device__ inline f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ inline uint32_t from_e4m3x2(uint32_t x, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, HI));
  }
};
template <> struct MatOp<f16_t> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static __device__ inline f32x4 mul(v8 a, v8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <bool HI>
  static __device__ inline uint32_t from_e4m3x2(uint32_t x, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, HI));
  }
};

// 8 entries (two dwords of 8-bit values) as a matrix operand
template <typename T>
__device__ inline typename MatOp<T>::v8 widen8(uint32_t a, uint32_t b, float scale) {
  const u32x4 w = {MatOp<T>::template from_e4m3x2<false>(a, scale),
                   MatOp<T>::template from_e4m3x2<true>(a, scale),
                   MatOp<T>::template from_e4m3x2<false>(b, scale),
                   MatOp<T>::template from_e4m3x2<true>(b, scale)};
  return __builtin_bit_cast(typename MatOp<T>::v8, w);
}

// x from lane ^ 16 and lane ^ 32, folded with max / sum: the four lanes of a row
__device__ inline float swap16(float x, int lane) {
  auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((lane & 16) ? s[0] : s[1]);
}
__device__ inline float swap32(float x, int lane) {
  auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((lane & 32) ? s[0] : s[1]);
}

template <typename T, bool E8, int D>
struct PagedGeom {
  static constexpr int CK = E8 ? 16 : 8;          // neighbouring keys of a lane
  static constexpr int STEP = 4 * CK;             // keys of a step
  static constexpr int KT = CK / 4;               // 16-key tiles of a step
  static constexpr int KL = E8 ? D / 64 : D / 32; // 16-byte loads of a key by a lane
  static constexpr int VL = D / 16;               // 16-byte loads of V by a lane
  static constexpr int U = CK / 8;                // P.V products' key groups of 32
  static constexpr int ES = E8 ? 1 : 2;
};

// One step's keys, as loaded.
template <typename T, bool E8, int D>
struct PagedStep {
  typedef PagedGeom<T, E8, D> G;
  u32x4 k[G::KT][G::KL];
  u32x4 v[G::VL];
  float ks, vs;
  int base;        // first key
  bool live;       // the page of this lane's CK keys exists
};

template <typename T, bool E8, int D, int R, bool ROWS, bool PIPE>
struct PagedWave {
  typedef PagedGeom<T, E8, D> G;
  typedef PagedStep<T, E8, D> Step;
  typedef typename std::conditional<E8, bf16_t, T>::type PT;   // what P and V multiply in
  typedef typename MatOp<T>::v8 Q8;
  typedef typename MatOp<PT>::v8 P8;

  const unsigned char* kp;    // this KV head's part of page 0
  const unsigned char* vp;
  const float* scales;
  const int32_t* table;
  int64_t page_stride;        // bytes of a page (all heads)
  int64_t num_pages;
  int Hkv, P, p_shift, slots;
  int lane, g, r;
  int lo, lim, minvis;        // keys [lo, lim); all rows that see any of them see [lo, minvis)
  float scale_log2;
  Q8 q[R][D / 32];
  f32x4 o[R][D / 16];
  float m[R], l[R];
  int vis[R];

  // the page of CK keys from `key` on (read as it is: checked by load)
  __device__ inline int32_t page_of(int key) const {
    const int s = key >> p_shift;
    return table[s < slots ? s : slots - 1];
  }
  __device__ inline void lookup(int base, int32_t* pk, int32_t* pv) const {
    *pk = page_of(base + ((r >> 2) * G::CK));
    *pv = page_of(base + g * G::CK);
  }
  __device__ inline void load(Step& st, int base, int32_t pk, int32_t pv) const {
    // K: this lane's key of tile t is chunk r / 4, key 4t + r % 4; V: chunk g, dim r
    const int kc = base + (r >> 2) * G::CK, vc = base + g * G::CK;
    const bool kok = kc < lim && pk >= 0 && pk < num_pages;
    const bool vok = vc < lim && pv >= 0 && pv < num_pages;
    // (page 0 stands in where there is none: what it gives is masked)
    const unsigned char* ka = kp + (kok ? (int64_t)pk : 0) * page_stride +
                              (((kc & (P - 1)) + (r & 3)) * D + g * (16 / G::ES)) * G::ES;
    const unsigned char* va = vp + (vok ? (int64_t)pv : 0) * page_stride +
                              (r * P + (vc & (P - 1))) * G::ES;
#pragma unroll
    for (int t = 0; t < G::KT; ++t)
#pragma unroll
      for (int i = 0; i < G::KL; ++i) st.k[t][i] = load16(ka + t * 4 * D * G::ES + i * 64);
    const int vrow = 16 * P * G::ES;
#pragma unroll
    for (int i = 0; i < G::VL; ++i) st.v[i] = load16(va + i * vrow);
    st.ks = st.vs = 1.0f;
    if constexpr (E8) {
      if (vok) {
        const float* sc = scales + (int64_t)pv * Hkv * 2;
        st.ks = sc[0];
        st.vs = sc[1];
      }
    }
    st.base = base;
    st.live = vok;
  }

  // V operand u of dims 16 i .. 16 i + 15
  __device__ inline P8 v_op(const u32x4& v, int u, float vs) const {
    if constexpr (E8)
      return u == 0 ? widen8<PT>(v.x, v.y, vs) : widen8<PT>(v.z, v.w, vs);
    else
      return __builtin_bit_cast(P8, v);
  }
  // v with the keys outside [a, b) of the lane's CK zeroed
  __device__ inline u32x4 keep(const u32x4& v, int a, int b) const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t x[4];
    constexpr int per = 4 / G::ES, bits = 8 * G::ES;   // entries of a dword
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int from = a - i * per, to = b - i * per;
      const uint32_t below = to <= 0 ? 0u : (to >= per ? 0xffffffffu : (1u << (to * bits)) - 1u);
      const uint32_t skip = from <= 0 ? 0u : (from >= per ? 0xffffffffu : (1u << (from * bits)) - 1u);
      x[i] = w[i] & below & ~skip;
    }
    return u32x4{x[0], x[1], x[2], x[3]};
  }
  // the top bit of every entry of a dword that is not finite
  __device__ inline uint32_t not_finite(uint32_t w) const {
    constexpr bool bf = std::is_same<T, bf16_t>::value;
    if constexpr (E8)
      return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    else
      return ((w & (bf ? 0x7f807f80u : 0x7c007c00u)) + (bf ? 0x00800080u : 0x04000400u)) & 0x80008000u;
  }
  __device__ inline bool not_finite(const u32x4& v) const {
    return (not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w)) != 0;
  }
  __device__ inline uint32_t finite_part(uint32_t w) const {
    return w & ~((not_finite(w) >> (8 * G::ES - 1)) * (E8 ? 0xffu : 0xffffu));
  }

  __device__ inline void fold(Step& st) {
    const int cb = st.base + g * G::CK;
    f32x4 s[R][G::KT];
#pragma unroll
    for (int t = 0; t < G::KT; ++t) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) s[rt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        Q8 a;
        if constexpr (E8) {
          const u32x4 w = st.k[t][j >> 1];
          a = (j & 1) ? widen8<T>(w.z, w.w, 1.0f) : widen8<T>(w.x, w.y, 1.0f);
        } else {
          a = __builtin_bit_cast(Q8, st.k[t][j]);
        }
#pragma unroll
        for (int rt = 0; rt < R; ++rt) s[rt][t] = MatOp<T>::mul(a, q[rt][j], s[rt][t]);
      }
    }
    const float c = E8 ? st.ks * scale_log2 : scale_log2;
    // every row sees all keys of the step, and their pages exist
    const bool whole = st.base + G::STEP <= minvis && __all(st.live);
    P8 hi[R][G::U], rest[R][G::U];
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const int n = whole ? G::CK : (st.live ? vis[rt] - cb : 0);   // keys of this lane's that the row sees
      float x[G::CK];
      float top = kNegBig;
#pragma unroll
      for (int e = 0; e < G::CK; ++e) {
        x[e] = s[rt][e >> 2][e & 3] * c;
        if (!whole) x[e] = e < n ? x[e] : -INFINITY;
        top = fmaxf(top, x[e]);
      }
      top = fmaxf(top, swap16(top, lane));
      top = fmaxf(top, swap32(top, lane));
      const float m_new = fmaxf(m[rt], top);
      const float alpha = fast_exp2(m[rt] - m_new);
      if (!__all(m_new == m[rt])) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[rt][i] *= alpha;
      }
      m[rt] = m_new;
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < G::U; ++u) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = fast_exp2(x[8 * u + e] - m_new);
          sum += p;
          const PT h = (PT)p;
          hi[rt][u][e] = h;
          rest[rt][u][e] = (PT)(p - (float)h);
        }
      }
      l[rt] = l[rt] * alpha + sum;
    }
    bool odd = false;
    if (!whole) {
      const int n = st.live ? lim - cb : 0;
#pragma unroll
      for (int i = 0; i < G::VL; ++i) st.v[i] = keep(st.v[i], 0, n);
      if (minvis < lim) {
        bool any = false;
#pragma unroll
        for (int i = 0; i < G::VL; ++i) any |= not_finite(st.v[i]);
        odd = __any(any);
        if (odd) {
#pragma unroll
          for (int i = 0; i < G::VL; ++i) {
            st.v[i].x = finite_part(st.v[i].x);
            st.v[i].y = finite_part(st.v[i].y);
            st.v[i].z = finite_part(st.v[i].z);
            st.v[i].w = finite_part(st.v[i].w);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
#pragma unroll
      for (int u = 0; u < G::U; ++u) {
        const P8 a = v_op(st.v[i], u, st.vs);
#pragma unroll
        for (int rt = 0; rt < R; ++rt) {
          o[rt][i] = MatOp<PT>::mul(a, hi[rt][u], o[rt][i]);
          o[rt][i] = MatOp<PT>::mul(a, rest[rt][u], o[rt][i]);
        }
      }
    }
    if (odd) add_not_finite(st.base);
  }

  // The entries of a step that are not finite, added to the rows that see their keys (the
  // products took them as 0: p * NaN is NaN for p = 0 too).  From memory, one key at a
  // time: a step that needs it is rare.  For a weight p > 0 the product is the entry.
  __device__ inline void add_not_finite(int base) {
    const int end = base + G::STEP < lim ? base + G::STEP : lim;
#pragma unroll 1
    for (int key = base; key < end; ++key) {
      const int32_t page = page_of(key);
      if (page < 0 || page >= num_pages) continue;
      const unsigned char* p = vp + page * page_stride + (4 * g * P + (key & (P - 1))) * G::ES;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned char* at = p + (16 * i + e) * P * G::ES;
          float v;
          if constexpr (E8)
            v = from_e4m3(*at);
          else
            v = Elem<T>::to_f32(*reinterpret_cast<const T*>(at));
          if (!(fabsf(v) <= 3.402823466e38f)) {
#pragma unroll
            for (int rt = 0; rt < R; ++rt) o[rt][i][e] += vis[rt] > key ? v : 0.0f;
          }
        }
      }
    }
  }
};

template <typename T, bool E8, int D, int R, bool ROWS, bool PIPE>
__global__ __launch_bounds__(256, D > 128 || (PIPE && R > 1) ? 1 : 2) void paged_attn_mfma_kernel(PagedAttnArgs a) {
  typedef PagedWave<T, E8, D, R, ROWS, PIPE> Wave;
  typedef PagedGeom<T, E8, D> G;
  typedef PagedStep<T, E8, D> Step;
  constexpr int kPitch = D + 4;                    // of a row in LDS: rows fall on different banks
  __shared__ float acc_s[ROWS ? 1 : 4 * 16 * R * kPitch];
  __shared__ float ml_s[ROWS ? 1 : 4 * 16 * R * 2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int blk = blockIdx.x;
  const int split = blk % a.splits; blk /= a.splits;
  const int hk = blk % a.Hkv, b = blk / a.Hkv;
  const int n_rows = a.S * a.group;                // rows of this KV head
  const int block_row = blockIdx.y * (ROWS ? 64 * R : 16 * R);
  const int row0 = ROWS ? block_row + wave * 16 * R : block_row;
  const RowKeys rk = row_keys(a, b);

  Wave w;
  w.lane = lane;
  w.g = lane >> 4;
  w.r = lane & 15;
  const int64_t head_bytes = (int64_t)a.P * D * G::ES;
  w.kp = static_cast<const unsigned char*>(a.kp) + hk * head_bytes;
  w.vp = static_cast<const unsigned char*>(a.vp) + hk * head_bytes;
  w.page_stride = head_bytes * a.Hkv;
  w.scales = E8 ? a.scales + 2 * hk : nullptr;
  w.table = a.table + (int64_t)b * a.t_sb;
  w.num_pages = a.num_pages;
  w.Hkv = a.Hkv; w.P = a.P; w.p_shift = a.p_shift; w.slots = a.slots;
  w.scale_log2 = a.scale_log2;

  // keys of the block: those its last row sees, this split's part of them
  auto last_vis = [&](int first, int count) {      // of rows [first, first + count)
    const int last = first + count < n_rows ? first + count : n_rows;
    if (first >= last) return 0;
    const int s_hi = (last - 1) / a.group;
    return rk.vis(s_hi < rk.n ? s_hi : (rk.n > 0 && first / a.group < rk.n ? rk.n - 1 : s_hi));
  };
  int hi;
  split_range(last_vis(block_row, ROWS ? 64 * R : 16 * R), split, a.splits, &w.lo, &hi);
  if (ROWS) {
    const int own = last_vis(row0, 16 * R);
    hi = own < hi ? own : hi;
  }
  w.lim = hi;
  w.minvis = row0 < n_rows ? rk.vis(row0 / a.group) : 0;
  w.minvis = w.minvis > w.lo ? w.minvis : w.lo;

#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    const int row = row0 + 16 * rt + w.r;
    const int s = row / a.group, hg = row - s * a.group;
    const bool real = row < n_rows;
    w.vis[rt] = real ? rk.vis(s) : 0;
    w.m[rt] = kNegBig;
    w.l[rt] = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) w.o[rt][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const T* qp = static_cast<const T*>(a.q) + b * a.q_sb + (hk * a.group + hg) * a.q_sh + s * a.q_ss;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      // the dims of K's operand j
      const int d = E8 ? (j >> 1) * 64 + w.g * 16 + (j & 1) * 8 : j * 32 + w.g * 8;
      typename Wave::Q8 x;
      if (!real) {
        x = __builtin_bit_cast(typename Wave::Q8, u32x4{0u, 0u, 0u, 0u});
      } else if (a.q_vec) {
        x = __builtin_bit_cast(typename Wave::Q8, load16(qp + d));
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = qp[d + e];
      }
      w.q[rt][j] = x;
    }
  }

  const int stride = ROWS ? G::STEP : 4 * G::STEP;
  int base = w.lo + (ROWS ? 0 : wave * G::STEP);
  if (base < hi) {
    int32_t pk, pv;
    if constexpr (PIPE) {
      Step x, y;
      w.lookup(base, &pk, &pv);
      w.load(x, base, pk, pv);
      w.lookup(base + stride, &pk, &pv);
      for (;;) {
        base += stride;
        const bool more = base < hi;
        if (more) {
          w.load(y, base, pk, pv);
          w.lookup(base + stride, &pk, &pv);
        }
        w.fold(x);
        if (!more) break;
        base += stride;
        const bool again = base < hi;
        if (again) {
          w.load(x, base, pk, pv);
          w.lookup(base + stride, &pk, &pv);
        }
        w.fold(y);
        if (!again) break;
      }
    } else {
      Step x;
      w.lookup(base, &pk, &pv);
      for (; base < hi; base += stride) {
        w.load(x, base, pk, pv);
        w.lookup(base + stride, &pk, &pv);
        w.fold(x);
      }
    }
  }
#pragma unroll
  for (int rt = 0; rt < R; ++rt) {
    w.l[rt] += swap16(w.l[rt], lane);
    w.l[rt] += swap32(w.l[rt], lane);
    if (w.vis[rt] == 0) {   // no query token (whole steps do not look at each row's keys)
      w.m[rt] = kNegBig;
      w.l[rt] = 0.0f;
    }
  }

  // where 4 dims from d of a row go
  auto put = [&](int row, int d, f32x4 v, float M, float L) {
    const int s = row / a.group, h = hk * a.group + row - s * a.group;
    if (a.splits > 1) {
      const int64_t at = (((int64_t)b * a.Hq + h) * a.S + s) * a.splits + split;
      *reinterpret_cast<f32x4*>(a.part_acc + at * D + d) = v;
      if (d == 0) {
        a.part_ml[2 * at] = M;
        a.part_ml[2 * at + 1] = L;
      }
      return;
    }
    T* op = static_cast<T*>(a.out) + b * a.o_sb + h * a.o_sh + s * a.o_ss + d;
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = L == 0.0f ? (T)0.0f : Elem<T>::from_f32(v[e] / L);
    if (a.o_vec) {
      *reinterpret_cast<t4*>(op) = y;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) op[e] = y[e];
    }
    if (d == 0 && a.lse != nullptr)
      a.lse[((int64_t)b * a.Hq + h) * a.S + s] = L == 0.0f ? -INFINITY : (M + fast_log2(L)) * kLn2;
  };

  if constexpr (ROWS) {
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const int row = row0 + 16 * rt + w.r;
      if (row < n_rows) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) put(row, 16 * i + 4 * w.g, w.o[rt][i], w.m[rt], w.l[rt]);
      }
    }
  } else {
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const int at = wave * 16 * R + 16 * rt + w.r;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<f32x4*>(acc_s + at * kPitch + 16 * i + 4 * w.g) = w.o[rt][i];
      if (w.g == 0) {
        ml_s[2 * at] = w.m[rt];
        ml_s[2 * at + 1] = w.l[rt];
      }
    }
    __syncthreads();
    for (int it = tid; it < 16 * R * (D / 4); it += 256) {
      const int rr = it / (D / 4), d = 4 * (it % (D / 4));
      if (block_row + rr >= n_rows) continue;
      float M = kNegBig, L = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) M = fmaxf(M, ml_s[2 * (i * 16 * R + rr)]);
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = i * 16 * R + rr;
        const float li = ml_s[2 * at + 1];
        if (li == 0.0f) continue;                  // the wave's keys are none of this row's
        const float f = fast_exp2(ml_s[2 * at] - M);
        L += f * li;
        v += f * *reinterpret_cast<const f32x4*>(acc_s + at * kPitch + d);
      }
      put(block_row + rr, d, v, M, L);
    }
  }
}

}  // namespace mi
