// Attention over a paged KV cache on the matrix cores: pages of the queries' type or of
// 8-bit floats, head_dim 64, 128 and 256.
//
// A wave holds R tiles of 16 query rows of one KV head (row = token * group + head of
// the group) and streams its keys from memory straight into matrix operands: nothing
// passes through LDS until the end.  Per step of 64 keys (8-bit pages), 32 or (fp32) 16:
//   S^T = K Q^T      v_mfma_f32_16x16x32: A = 16 keys x 32 dims, B = 32 dims x 16 rows.
//                    A lane's operand is 8 dims of one key; the order of the dims is
//                    free as long as Q has the same, so each lane takes whole 16-byte
//                    pieces of its key.
//   softmax          the accumulator gives lane (g, r) = (lane / 16, lane % 16) four
//                    keys of row r per tile.  Which key is which row of A is free too:
//                    tile t's row 4g + i is key g * CK + 4t + i (CK = 16, 8 or 4), so
//                    that lane (g, r) ends up with the CK neighbouring keys g * CK ..
//                    of row r, and the row's largest score is two lane swaps away.
//   O^T += V^T P^T   A = 16 dims x 32 keys, B = 32 keys x 16 rows.  P^T's lane (g, r)
//                    needs 8 keys of row r: those it already has (no shuffle), and
//                    V^T's lane the same 8 keys of one dim: 8 or 16 neighbouring entries
//                    of the transposed V page, one 16-byte load.
// 8-bit entries become bf16 (K, and with fp32 queries V: q's type) two at a time with v_cvt_scalef32_pk, exactly;
// V's page scale is the instruction's scale operand (bf16 has fp32's range, so no page
// overflows), K's multiplies the scores.  p goes in as a 16-bit value and its remainder
// (two products): off by 2^-16 at most, where one rounding of p to q's type would add an
// error as large as that of the output itself.  l sums p in fp32.  fp32 queries run on
// v_mfma_f32_16x16x4 in the same layout, 4 dims (keys) a lane, and p as it is.
//
// The block's 4 waves take every 4th step of its keys and join through LDS at the end.
//
// Blocks (parts > 0): the keys that the rows of the batch have, in units of 64, are one
// list for each KV head and tile of query rows, and each block takes an equal part of
// it: with lengths that differ 8-fold no block is longer than another.  A part that
// starts or ends inside a row leaves the row's sums in the workspace, at most two such
// per part, and paged_mfma_join_kernel adds them up.  Where no row is much longer than a
// part, or with parts = 0, a block takes a whole row instead.
//
// A load covers whole 128-byte lines where a key is one or more (a pair of loads takes
// half-lines of its own rows and of rows 8 away, and the lanes exchange them), and is
// non-temporal where no other block reads the same keys (64 rows of 4 tokens, 8-bit pages: 123
// us, 137 without; one row of 131072 bf16 keys 95 and 107).  A row of V longer than 64 bytes
// is taken by two waves or steps, half a line each, and stays in the caches for the second
// (16 rows, bf16, pages of 64: 64.1 us, non-temporal 64.6).
//
// What bounds it.  Up to 16 query rows a KV head: memory; with everything but the loads left
// out it takes 96 to 98 % of the time.  64 rows of 4 tokens, 24 heads over 8 of 128, up to
// 8192 8-bit keys: 614 MB in 115.6 us, 5.3 TB/s (a 4 GiB copy reaches 4.8); 16 rows of 1024 ..
// 8192 bf16 keys in pages of 16: 317 MB in 54.2 us, 5.9 TB/s; one row of 131072 8-bit keys: 268
// MB in 48.8 us, 5.5 TB/s.  The join of divided rows adds 5.6 to 7.8 us.  Pieces of prompts:
// the softmax's vector instructions and the two products of p (511 tokens over 4096 8-bit
// keys, 32 heads over 8 of 64: 43.6 us, 370 TFLOP/s of Q K and P V; without p's remainder
// 35), and with 16-bit pages the L1, which takes the loads 16 bytes a clock, a lane a row of
// the page (66 us).  Keys that the block's waves share in LDS are 1.1 to 1.5 times faster
// there from 512 tokens of 4096 keys or 4 rows of 512 on, and 1.1 to 2 times slower below.
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
  // a and b rounded, and their rounded values
  static __device__ inline uint32_t pack(float a, float b, float& ra, float& rb) {
    const uint32_t w = __builtin_bit_cast(uint32_t, v2{(__bf16)a, (__bf16)b});
    ra = __uint_as_float(w << 16);
    rb = __uint_as_float(w & 0xffff0000u);
    return w;
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
  static __device__ inline uint32_t pack(float a, float b, float& ra, float& rb) {
    const v2 w = {(_Float16)a, (_Float16)b};
    ra = (float)w[0];
    rb = (float)w[1];
    return __builtin_bit_cast(uint32_t, w);
  }
};

// fp32 operands are 4 dims (or keys) a lane, multiplied with v_mfma_f32_16x16x4 one by one
template <> struct MatOp<float> {
  typedef f32x4 v8;
  static __device__ inline f32x4 mul(v8 a, v8 b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// 4 8-bit entries (a dword) as an fp32 operand
__device__ inline f32x4 widen4(uint32_t x, float scale) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, scale, false);
  const f2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(x, scale, true);
  return f32x4{a[0], a[1], b[0], b[1]};
}

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
  static constexpr bool F32 = std::is_same<T, float>::value;
  static constexpr int ES = E8 ? 1 : (int)sizeof(T);
  static constexpr int CK = 16 / ES;              // neighbouring keys of a lane
  static constexpr int STEP = 4 * CK;             // keys of a step
  static constexpr int KT = CK / 4;               // 16-key tiles of a step
  static constexpr int KL = D * ES / 64;          // 16-byte loads of a key by a lane
  static constexpr bool PAIRS = KL % 2 == 0;      // a key is whole 128-byte lines
  static constexpr int VL = D / 16;               // 16-byte loads of V by a lane
  static constexpr int OE = F32 ? 4 : 8;          // dims (keys) of an operand that a lane holds
  static constexpr int NJ = D / (4 * OE);         // Q.K operands of a tile
  static constexpr int U = CK / OE;               // P.V operands of a step
};

// One step's keys and values, as loaded.
template <typename T, bool E8, int D>
struct PagedK {
  typedef PagedGeom<T, E8, D> G;
  u32x4 k[G::KT][G::KL];
  float scale;
};
template <typename T, bool E8, int D>
struct PagedV {
  typedef PagedGeom<T, E8, D> G;
  u32x4 v[G::VL];
  float scale;
};

// Whether K of the next step is loaded ahead: 16-bit pages at head_dim 128 (128 K keys 104 us,
// 112 without; 16 ragged rows 63.5 and 64.6).  8-bit pages need the registers for their
// conversions (64 rows of drafts 131 us ahead, 124 without), and at head_dim 64 a third
// wave a SIMD hides more (64 rows of 4096 keys 42.5 us ahead, 39.4 without).
template <typename T, bool E8, int D, int R>
struct PagedAhead {
  static constexpr bool value = sizeof(T) == 2 && !E8 && R == 1 && D == 128;
};

template <typename T, bool E8, int D, int R, bool STREAM>
struct PagedWave {
  typedef PagedGeom<T, E8, D> G;
  typedef PagedK<T, E8, D> KStep;
  typedef PagedV<T, E8, D> VStep;
  typedef typename std::conditional<E8 && !G::F32, bf16_t, T>::type PT;   // what P and V multiply in
  typedef typename MatOp<T>::v8 Q8;
  typedef typename MatOp<PT>::v8 P8;

  const unsigned char* kp;    // this KV head's part of page 0
  const unsigned char* vp;
  const float* scales;
  const int32_t* table;
  uint32_t page_stride;       // bytes of a page (all heads; the host checks that they fit)
  uint32_t num_pages;
  int Hkv, P, p_shift, slots;
  int lane, g, r;
  int lo, lim, minvis;        // keys [lo, lim); all rows that see any of them see [lo, minvis)
  bool v_once;                // a step takes whole lines of V
  float scale_log2;
  Q8 q[R][G::NJ];
  f32x4 o[R][D / 16];
  float m[R], l[R];
  bool huge;                  // a score beyond 2^26 was seen
  int vis[R];

  // the page of CK keys from `key` on (read as it is: checked by load)
  __device__ inline int32_t page_of(int key) const {
    const int s = key >> p_shift;
    return table[s < slots ? s : slots - 1];
  }
  // pages of the step's keys that this lane loads
  struct Pages {
    int32_t k0, k1, v;
  };
  __device__ inline Pages lookup(int base) const {
    Pages p;
    if constexpr (G::PAIRS) {
      p.k0 = page_of(base + ((r & 7) >> 2) * G::CK);
      p.k1 = page_of(base + (2 + ((r & 7) >> 2)) * G::CK);
    } else {
      p.k0 = p.k1 = page_of(base + (r >> 2) * G::CK);
    }
    p.v = page_of(base + g * G::CK);
    return p;
  }
  // where a page's chunk of CK keys lies; page 0 stands in where there is none (what it
  // gives is masked)
  __device__ inline bool chunk(int key, int32_t page, int64_t* at) const {
    const bool ok = key < lim && (uint32_t)page < num_pages;
    *at = (int64_t)((uint64_t)(ok ? (uint32_t)page : 0u) * page_stride);
    return ok;
  }
  __device__ inline u32x4 fetch(const unsigned char* p) const {
    return STREAM ? load16_stream(p) : load16(p);
  }
  __device__ inline float page_scale(int32_t page, bool ok, int which) const {
    if constexpr (E8) {
      if (ok) return scales[(uint64_t)(uint32_t)page * (uint32_t)(2 * Hkv) + which];
    }
    return 1.0f;
  }
  __device__ inline void load_k(KStep& st, int base, const Pages& pg) const {
    int64_t at;
    if constexpr (G::PAIRS) {
      // Two loads of a pair take rows 0..7 and 8..15 of the tile, lanes r < 8 the first and
      // r >= 8 the second 64 bytes of a 128-byte line: each load takes whole lines
      // (fold exchanges them).
      const int key0 = base + ((r & 7) >> 2) * G::CK, key1 = key0 + 2 * G::CK;
      const int in_line = (r >> 3) * 64 + g * 16;
      chunk(key0, pg.k0, &at);
      const unsigned char* k0 = kp + at + ((key0 & (P - 1)) + (r & 3)) * D * G::ES + in_line;
      chunk(key1, pg.k1, &at);
      const unsigned char* k1 = kp + at + ((key1 & (P - 1)) + (r & 3)) * D * G::ES + in_line;
#pragma unroll
      for (int t = 0; t < G::KT; ++t)
#pragma unroll
        for (int i = 0; i < G::KL; i += 2) {
          st.k[t][i] = fetch(k0 + t * 4 * D * G::ES + i * 64);
          st.k[t][i + 1] = fetch(k1 + t * 4 * D * G::ES + i * 64);
        }
    } else {
      const int key = base + (r >> 2) * G::CK;
      chunk(key, pg.k0, &at);
      const unsigned char* k0 = kp + at + ((key & (P - 1)) + (r & 3)) * D * G::ES + g * 16;
#pragma unroll
      for (int t = 0; t < G::KT; ++t) st.k[t][0] = fetch(k0 + t * 4 * D * G::ES);
    }
    st.scale = page_scale(pg.v, live(base, pg), 0);   // of the keys whose scores this lane gets
  }
  // the page of this lane's CK keys exists
  __device__ inline bool live(int base, const Pages& pg) const {
    return base + g * G::CK < lim && (uint32_t)pg.v < num_pages;
  }
  __device__ inline void load_v(VStep& st, int base, const Pages& pg) const {
    int64_t at;
    const int key = base + g * G::CK;
    const bool ok = chunk(key, pg.v, &at);
    const unsigned char* va = vp + at + (r * P + (key & (P - 1))) * G::ES;
#pragma unroll
    for (int i = 0; i < G::VL; ++i) st.v[i] = v_once ? fetch(va + i * 16 * P * G::ES) : load16(va + i * 16 * P * G::ES);
    st.scale = page_scale(pg.v, ok, 1);
  }
  // x for lanes of `banks` (0xc: r >= 8, 0x3: r < 8) from lane r ^ 8 of y
  template <int BANKS>
  static __device__ inline uint32_t from_other_half(uint32_t x, uint32_t y) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)y, 0x128, 0xf, BANKS, false);
  }
  // the 64-byte pieces of row r, from a pair of loads
  __device__ inline void exchange(u32x4& a, u32x4& b) const {
    const u32x4 x = a, y = b;
    a = u32x4{from_other_half<0xc>(x.x, y.x), from_other_half<0xc>(x.y, y.y),
              from_other_half<0xc>(x.z, y.z), from_other_half<0xc>(x.w, y.w)};
    b = u32x4{from_other_half<0x3>(y.x, x.x), from_other_half<0x3>(y.y, x.y),
              from_other_half<0x3>(y.z, x.z), from_other_half<0x3>(y.w, x.w)};
  }

  // the first dim of this lane in K operand j
  __device__ inline int dim_of(int j) const {
    if constexpr (!E8) return (j * 4 + g) * G::OE;
    constexpr int per = 16 / G::OE;                // operands of a 16-byte piece
    return j / per * 64 + g * 16 + j % per * G::OE;
  }
  // K operand j of tile t
  __device__ inline Q8 k_op(const KStep& st, int t, int j) const {
    if constexpr (E8 && G::F32) {
      return widen4(st.k[t][j >> 2][j & 3], 1.0f);
    } else if constexpr (E8) {
      const u32x4 w = st.k[t][j >> 1];
      return (j & 1) ? widen8<T>(w.z, w.w, 1.0f) : widen8<T>(w.x, w.y, 1.0f);
    } else {
      return __builtin_bit_cast(Q8, st.k[t][j]);
    }
  }
  // V operand u of dims 16 i .. 16 i + 15
  __device__ inline P8 v_op(const VStep& st, int i, int u) const {
    if constexpr (E8 && G::F32) {
      return widen4(st.v[i][u], st.scale);
    } else if constexpr (E8) {
      const u32x4 v = st.v[i];
      return u == 0 ? widen8<PT>(v.x, v.y, st.scale) : widen8<PT>(v.z, v.w, st.scale);
    } else {
      return __builtin_bit_cast(P8, st.v[i]);
    }
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
    else if constexpr (G::F32)
      return ((w & 0x7f800000u) + 0x00800000u) & 0x80000000u;
    else
      return ((w & (bf ? 0x7f807f80u : 0x7c007c00u)) + (bf ? 0x00800080u : 0x04000400u)) & 0x80008000u;
  }
  __device__ inline bool not_finite(const u32x4& v) const {
    return (not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w)) != 0;
  }
  __device__ inline uint32_t finite_part(uint32_t w) const {
    return w & ~((not_finite(w) >> (8 * G::ES - 1)) * (E8 ? 0xffu : G::F32 ? 0xffffffffu : 0xffffu));
  }

  P8 hi[R][G::U], rest[R][G::U];   // p of the step: its 16-bit value and the remainder (fp32: hi)
  bool whole, here;                // the step's keys are all seen by all rows; `live`

  // scores, softmax and p of the step at `base`
  __device__ inline void fold_k(KStep& st, int base, const Pages& pg) {
    const int cb = base + g * G::CK;
    here = live(base, pg);
    f32x4 s[R][G::KT];
    // two tiles at a time: products into one accumulator wait for each other
    constexpr int kTiles = G::KT < 2 ? G::KT : 2;
#pragma unroll
    for (int t0 = 0; t0 < G::KT; t0 += kTiles) {
      if constexpr (G::PAIRS) {
#pragma unroll
        for (int i = 0; i < G::KL; i += 2)
#pragma unroll
          for (int t = t0; t < t0 + kTiles; ++t) exchange(st.k[t][i], st.k[t][i + 1]);
      }
#pragma unroll
      for (int rt = 0; rt < R; ++rt)
#pragma unroll
        for (int t = t0; t < t0 + kTiles; ++t) s[rt][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < G::NJ; ++j) {
        Q8 k[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) k[t] = k_op(st, t0 + t, j);
#pragma unroll
        for (int rt = 0; rt < R; ++rt)
#pragma unroll
          for (int t = 0; t < kTiles; ++t) s[rt][t0 + t] = MatOp<T>::mul(k[t], q[rt][j], s[rt][t0 + t]);
      }
    }
    // (not below the least normal number: -inf times it must stay -inf)
    const float c = fmaxf(E8 ? st.scale * scale_log2 : scale_log2, 1.17549435e-38f);
    // every row sees all keys of the step, and their pages exist
    whole = base + G::STEP <= minvis && __all(here);
    if (!whole) {
#pragma unroll
      for (int rt = 0; rt < R; ++rt) {
        const int n = here ? vis[rt] - cb : 0;     // keys of this lane's that the row sees
#pragma unroll
        for (int e = 0; e < G::CK; ++e)
          s[rt][e >> 2][e & 3] = e < n ? s[rt][e >> 2][e & 3] : -INFINITY;
      }
      asm volatile("");   // (a branch: selects would cost every step)
    }
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      // the largest of the unscaled scores (the scale is positive and one for the lane's keys)
      float top = -INFINITY;
#pragma unroll
      for (int e = 0; e < G::CK; ++e) top = fmaxf(top, s[rt][e >> 2][e & 3]);
      top *= c;
      top = fmaxf(top, swap16(top, lane));
      top = fmaxf(top, swap32(top, lane));
      // the maximum moves only where p would pass 2^8: otherwise some row of the 16 moves it
      // in most steps (511 tokens of 8-bit pages, head_dim 64: 4096 keys 45.8 us, moved in
      // every step 47.3; 8192 keys 78.1 and 80.6)
      const bool over = top > m[rt] + 8.0f;
      if (__any(over)) {
        // Beyond 2^26 a score's rounding (2^-24 of it) passes the 2^2 that p's types bear: the
        // maximum is then taken below that, and p held to 1.
        const bool far = fabsf(top) > 67108864.0f;
        const float lower = fmaxf(top - fabsf(top) * 2.3841858e-07f, kLowest);
        const float m_new = over ? (far ? lower : top) : m[rt];
        huge |= __any(over && far) != 0;
        const float alpha = fast_exp2(m[rt] - m_new);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[rt][i] *= alpha;
        l[rt] *= alpha;
        m[rt] = m_new;
      }
      float scale = c, sub = m[rt];
      if (huge) {
#pragma unroll
        for (int e = 0; e < G::CK; ++e) {
          const float x = fmaf(s[rt][e >> 2][e & 3], c, -m[rt]);
          s[rt][e >> 2][e & 3] = x > 0.0f ? 0.0f : x;   // (a NaN stays)
        }
        scale = 1.0f;
        sub = 0.0f;
      }
      float sum = 0.0f;
#pragma unroll
      for (int u = 0; u < G::U; ++u) {
        if constexpr (G::F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            hi[rt][u][e] = fast_exp2(fmaf(s[rt][u][e], scale, -sub));
            sum += hi[rt][u][e];
          }
        } else {
          uint32_t h[4], x[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int k = 8 * u + 2 * e;
            const float p0 = fast_exp2(fmaf(s[rt][k >> 2][k & 3], scale, -sub));
            const float p1 = fast_exp2(fmaf(s[rt][k >> 2][(k & 3) + 1], scale, -sub));
            sum += p0 + p1;
            float h0, h1;
            h[e] = MatOp<PT>::pack(p0, p1, h0, h1);
            x[e] = MatOp<PT>::pack(p0 - h0, p1 - h1, h0, h1);
          }
          hi[rt][u] = __builtin_bit_cast(P8, u32x4{h[0], h[1], h[2], h[3]});
          rest[rt][u] = __builtin_bit_cast(P8, u32x4{x[0], x[1], x[2], x[3]});
        }
      }
      l[rt] += sum;
    }
  }

  // o += V^T P^T
  __device__ inline void fold_v(VStep& st, int base) {
    bool odd = false;
    if (!whole) {
      const int n = here ? lim - (base + g * G::CK) : 0;
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
    constexpr int kTogether = 2;   // dims' accumulators in turn, as above
#pragma unroll
    for (int i = 0; i < D / 16; i += kTogether) {
#pragma unroll
      for (int u = 0; u < G::U; ++u) {
        P8 a[kTogether];
#pragma unroll
        for (int j = 0; j < kTogether; ++j) a[j] = v_op(st, i + j, u);
#pragma unroll
        for (int rt = 0; rt < R; ++rt) {
#pragma unroll
          for (int j = 0; j < kTogether; ++j) o[rt][i + j] = MatOp<PT>::mul(a[j], hi[rt][u], o[rt][i + j]);
        }
        if constexpr (!G::F32) {
#pragma unroll
          for (int rt = 0; rt < R; ++rt) {
#pragma unroll
            for (int j = 0; j < kTogether; ++j) o[rt][i + j] = MatOp<PT>::mul(a[j], rest[rt][u], o[rt][i + j]);
          }
        }
      }
    }
    if (odd) add_not_finite(base);
  }

  // The entries of a step that are not finite, added to the rows that see their keys (the
  // products took them as 0: p * NaN is NaN for p = 0 too).  From memory, one key at a
  // time: a step that needs it is rare.  For a weight p > 0 the product is the entry.
  __device__ inline void add_not_finite(int base) {
    const int end = base + G::STEP < lim ? base + G::STEP : lim;
#pragma unroll 1
    for (int key = base; key < end; ++key) {
      const int32_t page = page_of(key);
      if ((uint32_t)page >= num_pages) continue;
      const unsigned char* p = vp + (int64_t)((uint64_t)page * page_stride) + (4 * g * P + (key & (P - 1))) * G::ES;
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

// ------------------------------------------------ the list of a KV head's keys
// Rows b = 0 .. B-1, each with ceil(vis / 64) units, vis the keys that the last query
// row of a tile sees.  A wave holds 64 rows of it at a time, one a lane.
struct UnitList {
  const PagedAttnArgs* a;
  int s_first, s_last;       // query tokens of the tile's first and last row
  int lane;
  int b0;                    // first row held
  int units, end;            // the lane's row: its units, and the list's up to it
  int before;                // units of the rows before b0
  int longest;               // most units of a row (after total())

  __device__ inline int vis_of(const RowKeys& rk) const {
    // the last query token that is real (tokens behind query_lens see nothing)
    return s_first < rk.n ? rk.vis(s_last < rk.n ? s_last : rk.n - 1) : 0;
  }
  __device__ inline void hold(int first, int units_before) {
    b0 = first;
    before = units_before;
    const int b = first + lane;
    units = b < a->B ? (vis_of(row_keys(*a, b)) + 63) >> 6 : 0;
    end = units;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
      const int x = __shfl_up(end, i, 64);
      if (lane >= i) end += x;
    }
    end += before;
  }
  __device__ inline int held_end() const { return __builtin_amdgcn_readlane(end, 63); }
  // the whole list's units; rows [0, 64) are held afterwards
  __device__ inline int total() {
    int t = 0, most = 0;
    for (int b = (a->B - 1) / 64 * 64; b > 0; b -= 64) {
      hold(b, 0);
      t += held_end();
      most = units > most ? units : most;
    }
    hold(0, 0);
    most = units > most ? units : most;
#pragma unroll
    for (int i = 32; i; i >>= 1) {
      const int x = __shfl_xor(most, i, 64);
      most = x > most ? x : most;
    }
    longest = __builtin_amdgcn_readfirstlane(most);
    return t + held_end();
  }
};
// parts in use (4 units each at least), and where part i of a list of `total` units starts
__device__ inline int parts_used(int total, int parts) {
  const int most = (total + 3) >> 2;
  return most < parts ? most : parts;
}
// part i takes q or, the first ones, q + 1 units of total = used * q + more
struct Parts {
  int used, q, more;
  __device__ inline Parts(int total, int parts) {
    used = parts_used(total, parts);
    q = used > 0 ? total / used : 0;
    more = total - q * used;
  }
  // Whether a block takes a row instead: no row is much longer than a part, so dividing
  // them would only cost the joins (256 rows of up to 1024 keys, head_dim 64: 37 us by row,
  // 53 in parts; 64 rows of up to 8192, head_dim 128: 134 and 124).
  __device__ inline bool by_row(int longest) const { return longest <= q + (q >> 2) + 8; }
  __device__ inline int start(int i) const { return i * q + (i < more ? i : more); }
  // the part that holds unit x
  __device__ inline int of(int x) const {
    const int longer = more * (q + 1);
    return x < longer ? x / (q + 1) : more + (x - longer) / q;
  }
};
// workspace: sums (D floats) and m, l of the two ends of each part
__device__ inline int64_t part_at(const PagedAttnArgs& a, int hk, int tile, int part, int end) {
  return ((((int64_t)hk * a.tiles + tile) * a.parts + part) * 2 + end) * a.kv_rows;
}

template <typename T>
__device__ inline void store_row4(const PagedAttnArgs& a, int b, int h, int s, int d, f32x4 v,
                                  float M, float L) {
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
}

template <typename T, bool E8, int D, int R, bool STREAM>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void paged_attn_mfma_kernel(PagedAttnArgs a) {
  typedef PagedWave<T, E8, D, R, STREAM> Wave;
  typedef PagedGeom<T, E8, D> G;
  constexpr int kRows = 16 * R;
  constexpr int kPitch = D + 4;                    // of a row in LDS: rows fall on different banks
  __shared__ float acc_s[4 * kRows * kPitch];
  __shared__ float ml_s[4 * kRows * 2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x % a.Hkv, part = blockIdx.x / a.Hkv, tile = blockIdx.y;
  const int n_rows = a.S * a.group;                // query rows of this KV head
  const int row0 = tile * kRows;
  const int last = (row0 + kRows < n_rows ? row0 + kRows : n_rows) - 1;

  UnitList list;
  list.a = &a;
  list.lane = lane;
  list.s_first = row0 / a.group;
  list.s_last = last / a.group;

  // this block's units [u, u1) and the row b that they start in, whose units start at row_u
  int b = part, u = 0, u1 = 0, row_u = 0;
  bool by_row = a.parts == 0;
  if (a.parts > 0) {
    const Parts parts(list.total(), a.parts);
    by_row = parts.by_row(list.longest);
    if (part >= (by_row ? a.B : parts.used)) return;
    u = parts.start(part);
    u1 = parts.start(part + 1);
  }
  if (!by_row) {
    while (list.held_end() <= u) list.hold(list.b0 + 64, list.held_end());
    const int at = (int)__builtin_ctzll(__ballot(list.end > u));
    b = list.b0 + at;
    row_u = __builtin_amdgcn_readlane(list.end, at) - __builtin_amdgcn_readlane(list.units, at);
  }
  const int u0 = u;

  Wave w;
  w.lane = lane;
  w.g = lane >> 4;
  w.r = lane & 15;
  const int64_t head_bytes = (int64_t)a.P * D * G::ES;
  w.kp = static_cast<const unsigned char*>(a.kp) + hk * head_bytes;
  w.vp = static_cast<const unsigned char*>(a.vp) + hk * head_bytes;
  w.page_stride = (uint32_t)(head_bytes * a.Hkv);
  w.scales = E8 ? a.scales + 2 * hk : nullptr;
  w.num_pages = (uint32_t)a.num_pages;
  w.Hkv = a.Hkv; w.P = a.P; w.p_shift = a.p_shift; w.slots = a.slots;
  w.scale_log2 = a.scale_log2;
  w.v_once = a.P * G::ES <= 64;

  for (;;) {
    const RowKeys rk = row_keys(a, b);
    const int vis = list.vis_of(rk);
    const int units = (vis + 63) >> 6;
    int hi = vis;
    bool whole = true;       // this block has all of the row's keys
    w.lo = 0;
    if (!by_row) {
      const int from = u - row_u, to = u1 - row_u < units ? u1 - row_u : units;
      whole = from == 0 && to == units;
      w.lo = from * 64;
      hi = to * 64 < vis ? to * 64 : vis;
    }
    w.lim = hi;
    w.minvis = rk.vis(list.s_first);
    w.minvis = w.minvis > w.lo ? w.minvis : w.lo;
    w.table = a.table + (int64_t)b * a.t_sb;
    w.huge = false;
    // page numbers first: they are on their way while q is loaded
    constexpr int kStride = 4 * G::STEP;
    int base = w.lo + wave * G::STEP;
    typename Wave::Pages pg = w.lookup(base), next = w.lookup(base + kStride);
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      const int row = row0 + 16 * rt + w.r;
      const int s = row / a.group, hg = row - s * a.group;
      const bool real = row < n_rows;
      w.vis[rt] = real ? rk.vis(s) : 0;
      w.m[rt] = kLowest;
      w.l[rt] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) w.o[rt][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      const T* qp =
          static_cast<const T*>(a.q) + b * a.q_sb + (hk * a.group + hg) * a.q_sh + s * a.q_ss;
#pragma unroll
      for (int j = 0; j < G::NJ; ++j) {
        const int d = w.dim_of(j);
        typename Wave::Q8 x;
        if (!real) {
          x = __builtin_bit_cast(typename Wave::Q8, u32x4{0u, 0u, 0u, 0u});
        } else if (a.q_vec) {
          x = __builtin_bit_cast(typename Wave::Q8, load16(qp + d));
        } else {
#pragma unroll
          for (int e = 0; e < G::OE; ++e) x[e] = qp[d + e];
        }
        w.q[rt][j] = x;
      }
    }

    if (base < hi) {
      typename Wave::VStep v;
      if constexpr (PagedAhead<T, E8, D, R>::value) {
        // K of the next step is on its way from before this step's products, V of the next
        // from behind them
        typename Wave::KStep ka, kb;
        w.load_k(ka, base, pg);
        w.load_v(v, base, pg);
        for (;;) {
          const bool more = base + kStride < hi;
          if (more) w.load_k(kb, base + kStride, next);
          w.fold_k(ka, base, pg);
          w.fold_v(v, base);
          if (!more) break;
          base += kStride;
          w.load_v(v, base, next);
          pg = next;
          next = w.lookup(base + kStride);
          const bool again = base + kStride < hi;
          if (again) w.load_k(ka, base + kStride, next);
          w.fold_k(kb, base, pg);
          w.fold_v(v, base);
          if (!again) break;
          base += kStride;
          w.load_v(v, base, next);
          pg = next;
          next = w.lookup(base + kStride);
        }
      } else {
        typename Wave::KStep k;
        for (; base < hi; base += kStride) {
          w.load_k(k, base, pg);
          w.load_v(v, base, pg);
          w.fold_k(k, base, pg);
          w.fold_v(v, base);
          pg = next;
          next = w.lookup(base + 2 * kStride);
        }
      }
    }

    // the block's waves, joined
#pragma unroll
    for (int rt = 0; rt < R; ++rt) {
      w.l[rt] += swap16(w.l[rt], lane);
      w.l[rt] += swap32(w.l[rt], lane);
      if (w.vis[rt] == 0) {   // no query token (whole steps do not look at each row's keys)
        w.m[rt] = kLowest;
        w.l[rt] = 0.0f;
      }
      const int at = wave * kRows + 16 * rt + w.r;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<f32x4*>(acc_s + at * kPitch + 16 * i + 4 * w.g) = w.o[rt][i];
      if (w.g == 0) {
        ml_s[2 * at] = w.m[rt];
        ml_s[2 * at + 1] = w.l[rt];
      }
    }
    __syncthreads();
    const int64_t slot = whole ? 0 : part_at(a, hk, tile, part, u == u0 ? 0 : 1);
    for (int it = tid; it < kRows * (D / 4); it += 256) {
      const int rr = it / (D / 4), d = 4 * (it % (D / 4));
      if (row0 + rr >= n_rows) continue;
      float M = kLowest, L = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) M = fmaxf(M, ml_s[2 * (i * kRows + rr)]);
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = i * kRows + rr;
        const float li = ml_s[2 * at + 1];
        if (li == 0.0f) continue;                  // the wave's keys are none of this row's
        const float f = fast_exp2(ml_s[2 * at] - M);
        L += f * li;
        v += f * *reinterpret_cast<const f32x4*>(acc_s + at * kPitch + d);
      }
      if (whole) {
        const int row = row0 + rr, s = row / a.group;
        store_row4<T>(a, b, hk * a.group + row - s * a.group, s, d, v, M, L);
      } else {
        *reinterpret_cast<f32x4*>(a.part_acc + (slot + rr) * D + d) = v;
        if (d == 0) {
          a.part_ml[2 * (slot + rr)] = M;
          a.part_ml[2 * (slot + rr) + 1] = L;
        }
      }
    }
    // the next row with keys
    if (by_row) break;
    u = row_u + units;
    if (u >= u1) break;
    __syncthreads();                               // LDS is written again
    while (list.held_end() <= u) list.hold(list.b0 + 64, list.held_end());
    const int at = (int)__builtin_ctzll(__ballot(list.end > u));
    b = list.b0 + at;
    row_u = u;
  }
}

// Rows whose keys several parts had: sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i
// over them.  Rows without keys become 0; all others are written already.  A block takes
// the query rows of one tile (or, where that leaves most of the GPU idle, one of
// them), D / 4 threads a part's sums (4 dims each): with up to 4 parts the groups take
// a query row each, else they share the parts of one (one row of 131072 keys: 56 us in all,
// 84 if a group took all parts).
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_mfma_join_kernel(PagedAttnArgs a) {
  constexpr int kGroups = 256 / (D / 4);
  __shared__ f32x4 acc_s[256];
  __shared__ float l_s[kGroups];
  const int tid = threadIdx.x, lane = tid & 63;
  int blk = blockIdx.x;
  const int hk = blk % a.Hkv; blk /= a.Hkv;
  const int tile = blk % a.tiles, b = blk / a.tiles;
  const int n_rows = a.S * a.group, row0 = tile * a.kv_rows;
  const int rows = row0 + a.kv_rows < n_rows ? a.kv_rows : n_rows - row0;
  UnitList list;
  list.a = &a;
  list.lane = lane;
  list.s_first = row0 / a.group;
  list.s_last = (row0 + rows - 1) / a.group;
  const Parts parts(list.total(), a.parts);
  if (parts.by_row(list.longest)) return;          // every row is written, the empty ones too
  while (list.b0 + 64 <= b) list.hold(list.b0 + 64, list.held_end());
  const int end = __builtin_amdgcn_readlane(list.end, b - list.b0);
  const int units = __builtin_amdgcn_readlane(list.units, b - list.b0);
  const int first_u = end - units;
  const int grp = tid / (D / 4), d = 4 * (tid % (D / 4));
  int i0 = 0, i1 = -1, end0 = 0;
  if (units > 0) {
    i0 = parts.of(first_u);
    i1 = parts.of(end - 1);
    if (i0 == i1) return;
    // (in part i0 the row is the last one, unless it starts with it; in the others the first)
    end0 = parts.start(i0) == first_u ? 0 : 1;
  }
  const bool share = i1 - i0 >= 4;
  for (int rr = blockIdx.y + (share ? 0 : (int)gridDim.y * grp); rr < rows;
       rr += (int)gridDim.y * (share ? 1 : kGroups)) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    float L = 0.0f, M = kLowest;
    for (int i = i0 + (share ? lane : 0); i <= i1; i += share ? 64 : 1)
      M = fmaxf(M, a.part_ml[2 * (part_at(a, hk, tile, i, i == i0 ? end0 : 0) + rr)]);
    if (share) {
#pragma unroll
      for (int i = 32; i; i >>= 1) M = fmaxf(M, __shfl_xor(M, i, 64));
    }
    // 4 parts' loads in flight at a time
    const int step = share ? kGroups : 1;
    for (int i = i0 + (share ? grp : 0); i <= i1; i += 4 * step) {
      float m[4], l[4];
      f32x4 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int p = i + j * step <= i1 ? i + j * step : i;
        const int64_t at = part_at(a, hk, tile, p, p == i0 ? end0 : 0) + rr;
        m[j] = a.part_ml[2 * at];
        l[j] = i + j * step <= i1 ? a.part_ml[2 * at + 1] : 0.0f;
        x[j] = *reinterpret_cast<const f32x4*>(a.part_acc + at * D + d);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = l[j] == 0.0f ? 0.0f : fast_exp2(m[j] - M);
        if (l[j] != 0.0f) v += f * x[j];             // (else the part's keys are none of this row's)
        L += f * l[j];
      }
    }
    if (share) {
      acc_s[tid] = v;
      if (d == 0) l_s[grp] = L;
      __syncthreads();
      if (grp == 0) {
        for (int i = 1; i < kGroups; ++i) {
          v += acc_s[tid + i * (D / 4)];
          L += l_s[i];
        }
      }
      __syncthreads();
    }
    if (!share || grp == 0) {
      const int row = row0 + rr, s = row / a.group;
      store_row4<T>(a, b, hk * a.group + row - s * a.group, s, d, v, M, L);
    }
  }
}

}  // namespace mi
