// What the kernels of the paged KV cache share: the 8-bit entries, their scale,
// and the checks of a cache's shape.
#pragma once

#include "common.hpp"

namespace mi {

// ------------------------------------------------- 8-bit entries (e4m3)
// OCP 8-bit floats: 1 sign, 4 exponent and 3 fraction bits, largest value 448,
// NaN 0x7f, no infinity; gfx950's conversions round to nearest even.  The callers
// keep |x| <= 448; an infinity becomes NaN here.
__device__ inline float e4m3_ready(float x) {
  return fabsf(x) <= 3.402823466e38f ? x : __builtin_nanf("");
}
__device__ inline uint32_t pack4_e4m3(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_ready(a), e4m3_ready(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_ready(c), e4m3_ready(d), w, true);
}
__device__ inline uint64_t pack8_e4m3(const float* x, float mult) {
  const uint64_t lo = pack4_e4m3(x[0] * mult, x[1] * mult, x[2] * mult, x[3] * mult);
  const uint64_t hi = pack4_e4m3(x[4] * mult, x[5] * mult, x[6] * mult, x[7] * mult);
  return lo | (hi << 32);
}
__device__ inline uint8_t to_e4m3(float x) {
  const float r = e4m3_ready(x);
  return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(r, r, 0, false) & 0xff);
}
__device__ inline float from_e4m3(uint8_t x) {
  return __builtin_amdgcn_cvt_f32_fp8((int)x, 0);
}

// The least power of two s >= 2^-120 with a <= 448 s (a finite, >= 0).  With
// a = m 2^k, 1 <= m < 2, and 448 = 1.75 * 2^8: s = 2^(k-8) if m <= 1.75, else 2^(k-7).
// From the bits: k is the exponent field and m > 1.75 is fraction bits > 0x600000.
// Its reciprocal is a power of two too, so dividing by s is exact.
__device__ inline float e4m3_scale(float a) {
  const uint32_t u = __float_as_uint(a);
  int e = (int)(u >> 23) - 127 - ((u & 0x7fffffu) > 0x600000u ? 7 : 8);
  e = e < -120 ? -120 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// ------------------------------------------------------------ host side
// Shapes of a call on a paged cache; MI_OK, or the status with its message set.
inline int32_t paged_check(const char* what, int64_t batch, int64_t n_heads, int64_t n_kv_heads,
                           int64_t seq_len, int64_t head_dim, int64_t num_pages,
                           int64_t page_size, int64_t slots, int32_t dtype, int32_t store,
                           const void* scales) {
  if (dtype != MI_DTYPE_BF16 && dtype != MI_DTYPE_F16 && dtype != MI_DTYPE_F32) {
    set_last_error("%s: unknown dtype code", what);
    return MI_ERR_INVALID;
  }
  if (store != MI_STORE_SAME && store != MI_STORE_E4M3) {
    set_last_error("%s: unknown store code", what);
    return MI_ERR_INVALID;
  }
  if (store == MI_STORE_E4M3 && scales == nullptr) {
    set_last_error("%s: 8-bit pages need their scales", what);
    return MI_ERR_INVALID;
  }
  if (batch < 0 || seq_len < 0 || n_heads <= 0 || n_kv_heads <= 0 || head_dim <= 0 ||
      num_pages <= 0 || slots <= 0) {
    set_last_error("%s: invalid shape", what);
    return MI_ERR_INVALID;
  }
  if (n_heads % n_kv_heads != 0) {
    set_last_error("%s: query heads (%lld) must be divisible by KV heads (%lld)", what,
                   (long long)n_heads, (long long)n_kv_heads);
    return MI_ERR_INVALID;
  }
  if (head_dim > 256) {
    set_last_error("%s: head_dim must be <= 256, got %lld", what, (long long)head_dim);
    return MI_ERR_UNSUPPORTED;
  }
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0) {
    set_last_error("%s: page_size must be 16, 32, 64, 128 or 256, got %lld", what,
                   (long long)page_size);
    return MI_ERR_UNSUPPORTED;
  }
  // 32-bit indexes: a row's positions, its tokens and the number of rows, heads and pages
  if (slots * page_size > INT32_MAX - 1024 || seq_len > (1 << 24) || batch > (1 << 24) ||
      n_heads > (1 << 16) || num_pages > INT32_MAX || slots > INT32_MAX / 256) {
    set_last_error("%s: size out of range", what);
    return MI_ERR_UNSUPPORTED;
  }
  return MI_OK;
}

}  // namespace mi
