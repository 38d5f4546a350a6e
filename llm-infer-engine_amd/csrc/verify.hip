// Verification of drafted tokens against the target's probabilities.
//
// With p_i = softmax(target[b, i] / T) and q_i = softmax(draft[b, i] / T) (without
// draft logits: the point mass of the drafted token), draft i is accepted iff
//   u[b, i] q_i(x_i) < p_i(x_i)
// and all before it were.  n = the number accepted.  The token after them is drawn
// from w = max(p_n - q_n, 0) where draft n was refused (from p_n if w is zero
// everywhere), from p_n where none was left to refuse: the least j with
//   w_0 + .. + w_j > r[b] (w_0 + .. + w_{V-1}).
// The accepted tokens and this one are then distributed as the target's own.  T = 0:
// draft i is accepted iff it is the target's largest logit (the least index of
// equals), and the token after is that of row n.
//
// A NaN logit counts as -inf, +inf as the largest finite value.
//
// The choice compares sums over the vocabulary with a given number: between two
// tokens the sums differ by one probability, 1e-5 and less in a flat row, which
// sums of fp32 shares do not resolve.  Sums that choose are therefore fp64, of
// shares good to 1e-9 of themselves (Shares below: a table of 32 powers of two and a
// short fp32 series for what is left).  u q < p alone only compares three numbers: the
// sums below its p and q are of fp32 shares (1e-6).
//
// `stats` reads every row that may matter once (chunks of 8184 or 2040 logits, each in
// its block's registers: largest value, its index, sum of fp32 shares relative to it).
// `decide`, one block a (row, chunk), joins the stats and decides; `weigh` sums w over
// each wave's pieces of a chunk; `pick`, one wave a row, finds the piece and in it the
// token.  Where w is p_n - q_n the two rows' sums have to be exact first: decide adds
// them up, and weigh is a launch of its own; without draft logits their sum is a common
// factor, and decide weighs itself.  T = 0 needs the first two only.
//
// 64 rows of up to 7 drafts, 128256 tokens, bf16: stats read 214 MB in 46 us, 4.6 TB/s, bound
// by memory (51 with each logit cleaned by itself instead of held to [-max, 0] after the
// difference); decide 18.9 us and weigh 19.2, bound by their 20 vector instructions a share;
// pick 7.8.  2 rows of 3 drafts: 4.3, 6.2, 4.8 and 6.8 us, each a launch and a chain of dependent
// reads.  (pick as the work of a row's last block instead: the fence that shows it the
// others' sums writes back the L2 for every block, 106 us in all against 97; with sums that pass
// the L2 instead, 92 and 92, and 19.2 against 18.5 for 16 rows without draft logits.)
#include <algorithm>

#include "common.hpp"

namespace mi {

constexpr int kVMaxDrafts = 128;

struct VerifyArgs {
  const void* target;
  const void* draft;
  const int64_t* drafted;
  const float* u;
  const float* r;
  const int64_t* lens;
  int64_t* tokens;
  int64_t* accepted;
  // workspace: stats of each (b, row, chunk), rows = S + 1 target rows, S draft rows
  float* sums;
  float* tops;
  int32_t* args;
  double* wsum;       // [B, chunks, pieces, 2]: sums of w and of p
  double* zsum;       // [B, chunks, 2]: sums of shares of row n, of the target and of the draft
  double* fin;        // [B, 4]: largest value and 1 / sum of row n, of the target and of the draft
  int64_t t_sb, t_ss, d_sb, d_ss, x_sb, x_ss, u_sb, u_ss;
  int64_t V;
  double c;           // log2(e) / T
  int32_t B, S, rows, chunks, greedy;
};

// Shares 2^((x - m) c) of logits x <= m.  y = (x - m) c in fp64, held to [-1100, 0] (a NaN or
// -inf is then 0 in the end, +inf the largest); y = k / 32 + f, |f| <= 1/64, k from the low
// bits of y + 1.5 * 2^47; 2^(k/32) is a table entry times 2^(k/32's whole part), 2^f =
// 1 + f p(f) with p the series of ln 2 (f ln 2)^i / (i+1)! in fp32, off by 2^-24 of 0.011.
// The table's 32 doubles lie on all 64 LDS banks once: no lanes collide.
struct Shares {
  const double* table;      // LDS: 2^(i/32)
  double c, least;          // scale, the least x - m
  float m;
  __device__ inline void set(const double* t, float top, double scale) {
    table = t;
    m = top;
    c = scale;
    least = -1100.0 / scale;
  }
  __device__ inline double of(float x) const {
    const double magic = 211106232532992.0;         // 1.5 * 2^47
    const double d = fmin(fmax((double)x - (double)m, least), 0.0), z = fma(d, c, magic);
    const int k = (int)__double_as_longlong(z);
    const float f = (float)fma(d, c, magic - z);
    float p = 0.009618129f;                           // (ln 2)^4 / 4!
    p = fmaf(p, f, 0.05550411f);                      // (ln 2)^3 / 3!
    p = fmaf(p, f, 0.24022651f);                      // (ln 2)^2 / 2!
    p = fmaf(p, f, 0.69314718f);
    p *= f;
    const double t = table[k & 31];
    return ldexp(fma(t, (double)p, t), k >> 5);
  }
};
__device__ inline void fill_table(double* t) {
  if (threadIdx.x < 32) t[threadIdx.x] = exp2((double)threadIdx.x / 32.0);
}

__device__ inline float logit(float x) {
  return x != x ? -INFINITY : fminf(x, 3.402823466e38f);
}

__device__ inline int drafts_of(const VerifyArgs& a, int b) {
  const int64_t n = a.lens != nullptr ? a.lens[b] : a.S;
  return (int)(n < 0 ? 0 : (n > a.S ? a.S : n));
}

template <typename T>
__device__ inline const T* row_of(const VerifyArgs& a, int b, int row) {
  return row <= a.S
             ? reinterpret_cast<const T*>(a.target) + b * a.t_sb + row * a.t_ss
             : reinterpret_cast<const T*>(a.draft) + b * a.d_sb + (row - a.S - 1) * a.d_ss;
}

// The thread's E logits of a chunk: groups of 16 bytes aligned in memory, dealt to
// the threads in turn; places outside the chunk's [lo, hi) hold -inf.
template <typename T, int E>
struct ChunkLogits {
  static constexpr int N = Chunk<T>::kN;       // logits of a group
  static constexpr int G = E / N;              // groups of a thread
  static constexpr int kPieces = 4 * G;        // a wave's logits of one g: 64 N in a row
  // places of a chunk: with a group's misalignment they still fit the threads
  static constexpr int64_t kPlaces = 256 * E - 8;
  float x[E];
  int64_t base;                                // place of group 0's first logit (may be < lo)
  __device__ inline int64_t place(int g) const { return base + ((int64_t)g * 256 + threadIdx.x) * N; }
  __device__ inline void load(const T* row, int64_t lo, int64_t hi) {
    base = first_place(row, lo);
    load_places(row, lo, hi);
  }
  // the chunk starts at the group that holds lo
  static __device__ inline int64_t first_place(const T* row, int64_t lo) {
    return lo - (int64_t)(((uintptr_t)(row + lo) % 16) / sizeof(T));
  }
  // the logits at base's places (base may be another row's: groups are then not aligned)
  __device__ inline void load_places(const T* row, int64_t lo, int64_t hi) {
    const bool aligned = (uintptr_t)(row + base) % 16 == 0;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int64_t j = place(g);
      if (aligned && j >= lo && j + N <= hi) {
        Chunk<T>::unpack(load16(row + j), x + g * N);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          x[g * N + e] = j + e >= lo && j + e < hi ? Elem<T>::to_f32(row[j + e]) : -INFINITY;
      }
    }
  }
};

template <typename T, int E>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ float top_s[4];
  __shared__ int64_t at_s[4];
  __shared__ float sum_s[4];
  const int chunk = blockIdx.x, row = blockIdx.y % a.rows, b = blockIdx.y / a.rows;
  const int n = drafts_of(a, b);
  if (row <= a.S ? row > n : row - a.S - 1 >= n) return;   // no draft there
  const int64_t lo = chunk * ChunkLogits<T, E>::kPlaces;
  const int64_t hi = lo + ChunkLogits<T, E>::kPlaces < a.V ? lo + ChunkLogits<T, E>::kPlaces : a.V;
  ChunkLogits<T, E> c;
  c.load(row_of<T>(a, b, row), lo, hi);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < E; ++i) top = __builtin_amdgcn_fmed3f(c.x[i], top, INFINITY);   // (not of a NaN)
  top = logit(top);
  // least place of the thread's largest logit (T = 0): its places grow with i
  int64_t at = lo;
  if (a.greedy && top > -INFINITY) {
#pragma unroll
    for (int i = E - 1; i >= 0; --i)
      if (logit(c.x[i]) == top) at = c.place(i / c.N) + i % c.N;
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const float t2 = __shfl_xor(top, m, 64);
    const int64_t a2 = __shfl_xor((long long)at, m, 64);
    at = t2 > top ? a2 : (t2 == top && a2 < at ? a2 : at);
    top = fmaxf(top, t2);
  }
  const int wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    top_s[wave] = top;
    at_s[wave] = at;
  }
  __syncthreads();
  top = top_s[0];
  at = at_s[0];
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    const float t2 = top_s[w];
    const int64_t a2 = at_s[w];
    at = t2 > top ? a2 : (t2 == top && a2 < at ? a2 : at);
    top = fmaxf(top, t2);
  }
  float sum = 0.0f;
  if (!a.greedy && top > -INFINITY) {
    const float c32 = (float)a.c;
#pragma unroll
    for (int i = 0; i < E; ++i)
      sum += fast_exp2(__builtin_amdgcn_fmed3f(c.x[i] - top, -3.402823466e38f, 0.0f) * c32);
#pragma unroll
    for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m, 64);
  }
  if ((threadIdx.x & 63) == 0) sum_s[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int64_t i = (int64_t)blockIdx.y * a.chunks + chunk;
    a.tops[i] = top;
    a.args[i] = (int32_t)at;
    a.sums[i] = (sum_s[0] + sum_s[1]) + (sum_s[2] + sum_s[3]);
  }
}

// w and p of one logit pair of row n
struct Weights {
  Shares t, d;
  double zt, zd;
  bool refused, model;
  int64_t point;      // the drafted token of a refused draft without logits, else -1
  __device__ inline void get(float xt, float xd, int64_t j, double* w, double* p) const {
    *p = t.m == -INFINITY ? 0.0 : t.of(xt) * zt;
    double q = 0.0;
    if (refused) q = !model ? (j == point ? 1.0 : 0.0) : (d.m == -INFINITY ? 0.0 : d.of(xd) * zd);
    const double left = *p - q;
    *w = left > 0.0 ? left : 0.0;
  }
};

// w and p summed over each wave's pieces of a chunk of row k
template <typename T, int E>
__device__ inline void weigh_chunk(const VerifyArgs& a, const Weights& w, int b, int k, int chunk) {
  const int64_t lo = chunk * ChunkLogits<T, E>::kPlaces;
  const int64_t hi = lo + ChunkLogits<T, E>::kPlaces < a.V ? lo + ChunkLogits<T, E>::kPlaces : a.V;
  ChunkLogits<T, E> ct, cd;
  ct.load(row_of<T>(a, b, k), lo, hi);
  const bool pair = w.refused && w.model;
  if (pair) {
    cd.base = ct.base;
    cd.load_places(row_of<T>(a, b, a.S + 1 + k), lo, hi);
  }
  double* out = a.wsum + 2 * ((int64_t)b * a.chunks + chunk) * ct.kPieces;
#pragma unroll
  for (int g = 0; g < ct.G; ++g) {
    double ws = 0.0, ps = 0.0;
#pragma unroll
    for (int e = 0; e < ct.N; ++e) {
      const int i = g * ct.N + e;
      double wj, pj;
      w.get(ct.x[i], pair ? cd.x[i] : -INFINITY, ct.place(g) + e, &wj, &pj);
      ws += wj;
      ps += pj;
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      ws += __shfl_xor(ws, m, 64);
      ps += __shfl_xor(ps, m, 64);
    }
    if ((threadIdx.x & 63) == 0) {
      out[2 * (4 * g + (threadIdx.x >> 6))] = ws;
      out[2 * (4 * g + (threadIdx.x >> 6)) + 1] = ps;
    }
  }
}

// a chunk's sum of shares of one row, of this thread
template <typename T, int E>
__device__ inline double chunk_sum(const Shares& sh, const T* row, int64_t lo, int64_t hi) {
  if (sh.m == -INFINITY) return 0.0;
  ChunkLogits<T, E> c;
  c.load(row, lo, hi);
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < E; ++i) sum += sh.of(c.x[i]);
  return sum;
}

template <typename T, int E, bool MODEL>
__global__ __launch_bounds__(256) void verify_decide_kernel(VerifyArgs a) {
  __shared__ float top_s[2 * kVMaxDrafts + 1];
  __shared__ float inv_s[2 * kVMaxDrafts + 1];
  __shared__ int32_t arg_s[2 * kVMaxDrafts + 1];
  __shared__ int first_s;
  __shared__ double table[32], zt_s[4], zd_s[4];
  const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = drafts_of(a, b);
  if (!a.greedy) fill_table(table);
  if (tid == 0) first_s = n;
  // the drafted tokens and their logits, while the stats come
  const int64_t x = tid < n ? a.drafted[b * a.x_sb + tid * a.x_ss] : -1;
  const bool token = x >= 0 && x < a.V;
  float xt = -INFINITY, xd = -INFINITY, u = 1.0f;
  if (token && !a.greedy) {
    xt = logit(Elem<T>::to_f32(row_of<T>(a, b, tid)[x]));
    if (MODEL) xd = logit(Elem<T>::to_f32(row_of<T>(a, b, a.S + 1 + tid)[x]));
    u = a.u[b * a.u_sb + tid * a.u_ss];
  }
  // 16 lanes join a row's chunks
  const int l16 = tid & 15;
  const float c32 = (float)a.c;
  for (int row = tid >> 4; row < a.rows; row += 16) {
    if (row <= a.S ? row > n : row - a.S - 1 >= n) continue;
    const int64_t i = ((int64_t)b * a.rows + row) * a.chunks;
    float top = -INFINITY, z = 0.0f;   // z relative to the lane's top
    int32_t at = INT32_MAX;
    for (int c0 = l16; c0 < a.chunks; c0 += 64) {   // four reads in flight
      float ts[4], ss[4];
      int32_t as[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = c0 + 16 * j < a.chunks;
        const int c = in ? c0 + 16 * j : c0;
        ts[j] = a.tops[i + c];
        ss[j] = a.sums[i + c];
        as[j] = a.args[i + c];
        ts[j] = in ? ts[j] : -INFINITY;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float t = ts[j];
        if (t == -INFINITY) continue;
        if (t > top) {
          z = z * fast_exp2((top - t) * c32) + ss[j];
          top = t;
          at = as[j];
        } else {
          z += ss[j] * fast_exp2((t - top) * c32);
        }
      }
    }
    float all = top;
#pragma unroll
    for (int m = 8; m; m >>= 1) {
      const float t2 = __shfl_xor(all, m, 16);
      const int32_t a2 = __shfl_xor(at, m, 16);
      at = t2 > all ? a2 : (t2 == all && a2 < at ? a2 : at);
      all = fmaxf(all, t2);
    }
    z = top == -INFINITY ? 0.0f : z * fast_exp2((top - all) * c32);
#pragma unroll
    for (int m = 8; m; m >>= 1) z += __shfl_xor(z, m, 16);
    if (l16 == 0) {
      top_s[row] = all;
      arg_s[row] = all == -INFINITY ? -1 : at;
      inv_s[row] = z > 0.0f ? 1.0f / z : 0.0f;
    }
  }
  __syncthreads();
  if (tid < n) {
    bool ok = false;
    if (token && a.greedy) {
      ok = x == arg_s[tid];
    } else if (token && top_s[tid] > -INFINITY) {
      Shares sh;
      sh.set(table, top_s[tid], a.c);
      const double p = sh.of(xt) * inv_s[tid];
      double q = 1.0;
      if (MODEL) {
        const int dr = a.S + 1 + tid;
        sh.set(table, top_s[dr], a.c);
        q = top_s[dr] == -INFINITY ? 0.0 : sh.of(xd) * inv_s[dr];
      }
      ok = (double)u * q < p;
    }
    if (!ok) atomicMin(&first_s, tid);
  }
  __syncthreads();
  const int k = first_s;                       // drafts accepted
  if (chunk == 0) {
    for (int i = tid; i <= a.S; i += 256) {
      int64_t t = -1;
      if (i < k) t = a.drafted[b * a.x_sb + i * a.x_ss];
      if (i == k && a.greedy) t = arg_s[k];
      if (i != k || a.greedy) a.tokens[(int64_t)b * (a.S + 1) + i] = t;
    }
    if (tid == 0) a.accepted[b] = k;
  }
  if (a.greedy) return;
  const bool refused = k < n;
  const int dr_row = a.S + 1 + k;
  Weights w;
  w.refused = refused;
  w.model = MODEL;
  w.t.set(table, top_s[k], a.c);
  w.d.set(table, MODEL && refused ? top_s[dr_row] : -INFINITY, a.c);
  w.zt = inv_s[k];
  w.zd = 0.0;
  w.point = !MODEL && refused ? a.drafted[b * a.x_sb + k * a.x_ss] : -1;
  if (chunk == 0 && tid == 0) {
    double* f = a.fin + 4 * (int64_t)b;
    f[0] = w.t.m;
    f[1] = w.zt;
    f[2] = w.d.m;
    f[3] = 0.0;
  }
  if constexpr (!MODEL) {
    weigh_chunk<T, E>(a, w, b, k, chunk);
  } else {
    const int64_t lo = chunk * ChunkLogits<T, E>::kPlaces;
    const int64_t hi = lo + ChunkLogits<T, E>::kPlaces < a.V ? lo + ChunkLogits<T, E>::kPlaces : a.V;
    double zt = chunk_sum<T, E>(w.t, row_of<T>(a, b, k), lo, hi), zd = 0.0;
    if (refused) zd = chunk_sum<T, E>(w.d, row_of<T>(a, b, dr_row), lo, hi);
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      zt += __shfl_xor(zt, m, 64);
      zd += __shfl_xor(zd, m, 64);
    }
    if ((tid & 63) == 0) {
      zt_s[tid >> 6] = zt;
      zd_s[tid >> 6] = zd;
    }
    __syncthreads();
    if (tid < 2) {
      const double* z = tid == 0 ? zt_s : zd_s;
      a.zsum[2 * ((int64_t)b * a.chunks + chunk) + tid] = (z[0] + z[1]) + (z[2] + z[3]);
    }
  }
}

template <typename T, int E>
__global__ __launch_bounds__(256) void verify_weigh_kernel(VerifyArgs a) {
  __shared__ double table[32];
  const int chunk = blockIdx.x, b = blockIdx.y, lane = threadIdx.x & 63;
  fill_table(table);
  const int n = drafts_of(a, b), k = (int)a.accepted[b];
  double* f = a.fin + 4 * (int64_t)b;
  double zt = 0.0, zd = 0.0;
  for (int c = lane; c < a.chunks; c += 64) {
    zt += a.zsum[2 * ((int64_t)b * a.chunks + c)];
    zd += a.zsum[2 * ((int64_t)b * a.chunks + c) + 1];
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    zt += __shfl_xor(zt, m, 64);
    zd += __shfl_xor(zd, m, 64);
  }
  __syncthreads();
  Weights w;
  w.refused = k < n;
  w.model = true;
  w.t.set(table, (float)f[0], a.c);
  w.d.set(table, (float)f[2], a.c);
  w.zt = zt > 0.0 ? 1.0 / zt : 0.0;
  w.zd = zd > 0.0 ? 1.0 / zd : 0.0;
  w.point = -1;
  weigh_chunk<T, E>(a, w, b, k, chunk);
}

// inclusive sums over the wave's lanes
__device__ inline double wave_scan(double x, int lane) {
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const double y = __shfl_up(x, i, 64);
    if (lane >= i) x += y;
  }
  return x;
}

// One wave a row.  The pieces' sums, a run of them for each lane, lead to the piece in
// which the sum passes the goal; its 64 N logits, N a lane, to the token.  (Should
// rounding pass the goal nowhere, the last place with mass is taken.)
template <typename T, int E>
__global__ __launch_bounds__(64) void verify_pick_kernel(VerifyArgs a) {
  typedef ChunkLogits<T, E> C;
  __shared__ double table[32];
  const int b = blockIdx.x, lane = threadIdx.x;
  fill_table(table);
  __syncthreads();
  const int n = drafts_of(a, b), k = (int)a.accepted[b];
  const int64_t n_pieces = (int64_t)a.chunks * C::kPieces;
  const double* sums = a.wsum + 2 * (int64_t)b * n_pieces;
  const int64_t per = (n_pieces + 63) / 64;
  const int64_t i0 = lane * per < n_pieces ? lane * per : n_pieces;
  const int64_t i1 = i0 + per < n_pieces ? i0 + per : n_pieces;
  double ws = 0.0, ps = 0.0;
  for (int64_t i = i0; i < i1; ++i) {
    ws += sums[2 * i];
    ps += sums[2 * i + 1];
  }
  const double ws_end = wave_scan(ws, lane), ps_end = wave_scan(ps, lane);
  const double total_w = __shfl(ws_end, 63, 64), total_p = __shfl(ps_end, 63, 64);
  // w, or p itself where w is zero everywhere (where nothing was refused w is p)
  const bool use_w = total_w > 0.0;
  const double total = use_w ? total_w : total_p;
  int64_t* out = a.tokens + (int64_t)b * (a.S + 1) + k;
  if (!(total > 0.0)) {                        // a row without mass: no token
    if (lane == 0) *out = -1;
    return;
  }
  const double goal = (double)a.r[b] * total;
  const double mine = use_w ? ws : ps, mine_end = use_w ? ws_end : ps_end;
  uint64_t over = __ballot(mine > 0.0 && mine_end > goal);
  if (over == 0) over = 1ull << (63 - __builtin_clzll(__ballot(mine > 0.0)));
  const int who = (int)__builtin_ctzll(over);
  int64_t piece = -1;
  double below = 0.0;
  if (lane == who) {
    double run = mine_end - mine;
    for (int64_t i = i0; i < i1; ++i) {
      const double x = sums[2 * i + (use_w ? 0 : 1)];
      if (x > 0.0) {
        piece = i;
        below = run;
        if (run + x > goal) break;
      }
      run += x;
    }
  }
  piece = __shfl((long long)piece, who, 64);
  below = __shfl(below, who, 64);

  Weights w;
  const double* f = a.fin + 4 * (int64_t)b;
  w.refused = k < n;
  w.model = a.draft != nullptr;
  w.t.set(table, (float)f[0], a.c);
  w.d.set(table, (float)f[2], a.c);
  w.zt = f[1];
  w.zd = 0.0;
  if (w.model) {                               // as weigh had them
    double zt = 0.0, zd = 0.0;
    for (int c = lane; c < a.chunks; c += 64) {
      zt += a.zsum[2 * ((int64_t)b * a.chunks + c)];
      zd += a.zsum[2 * ((int64_t)b * a.chunks + c) + 1];
    }
#pragma unroll
    for (int m = 32; m; m >>= 1) {
      zt += __shfl_xor(zt, m, 64);
      zd += __shfl_xor(zd, m, 64);
    }
    w.zt = zt > 0.0 ? 1.0 / zt : 0.0;
    w.zd = zd > 0.0 ? 1.0 / zd : 0.0;
  }
  w.point = w.refused && !w.model ? a.drafted[b * a.x_sb + k * a.x_ss] : -1;
  const T* tr = row_of<T>(a, b, k);
  const T* dr = w.refused && w.model ? row_of<T>(a, b, a.S + 1 + k) : nullptr;
  const int64_t lo = piece / C::kPieces * C::kPlaces;
  const int64_t hi = lo + C::kPlaces < a.V ? lo + C::kPlaces : a.V;
  const int64_t j0 = C::first_place(tr, lo) + (piece % C::kPieces * 64 + lane) * C::N;
  double x[C::N], sum = 0.0;
#pragma unroll
  for (int e = 0; e < C::N; ++e) {
    const int64_t j = j0 + e;
    x[e] = 0.0;
    if (j >= lo && j < hi) {
      double wj, pj;
      w.get(Elem<T>::to_f32(tr[j]), dr != nullptr ? Elem<T>::to_f32(dr[j]) : -INFINITY, j, &wj, &pj);
      x[e] = use_w ? wj : pj;
    }
    sum += x[e];
  }
  double run = below + wave_scan(sum, lane) - sum;
  int64_t hit = INT64_MAX, last = -1;
#pragma unroll
  for (int e = 0; e < C::N; ++e) {
    run += x[e];
    if (x[e] > 0.0) {
      last = j0 + e;
      if (run > goal && hit == INT64_MAX) hit = j0 + e;
    }
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) {
    const int64_t h = __shfl_xor((long long)hit, m, 64), l = __shfl_xor((long long)last, m, 64);
    hit = h < hit ? h : hit;
    last = l > last ? l : last;
  }
  if (lane == 0) *out = hit != INT64_MAX ? hit : last;
}

namespace {

// Logits of a thread: 32, or 8 where chunks of 32 leave most of the GPU idle
// (2 rows of 3 drafts, 128256 tokens: 25.8 us with 8, 33.6 with 32).
int verify_elems(int64_t batch, int64_t vocab) {
  return batch * ((vocab + 8183) / 8184) < device_cu_count() ? 8 : 32;
}
int64_t verify_chunks(int64_t vocab, int elems) {
  const int64_t places = 256 * (int64_t)elems - 8;
  return (vocab + places - 1) / places;
}
// pieces of the chunks: elems / 2 of a chunk for 2-byte logits, elems for fp32
int64_t verify_pieces(int64_t vocab, int elems) { return verify_chunks(vocab, elems) * elems; }
int64_t up8(int64_t bytes) { return (bytes + 7) / 8 * 8; }

template <typename T, int E>
void launch_verify(const VerifyArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((verify_stats_kernel<T, E>), dim3(a.chunks, a.B * a.rows), dim3(256), 0, st, a);
  const dim3 grid(a.greedy ? 1 : a.chunks, a.B);
  if (a.draft != nullptr) {
    hipLaunchKernelGGL((verify_decide_kernel<T, E, true>), grid, dim3(256), 0, st, a);
    hipLaunchKernelGGL((verify_weigh_kernel<T, E>), grid, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((verify_decide_kernel<T, E, false>), grid, dim3(256), 0, st, a);
  }
  if (!a.greedy)
    hipLaunchKernelGGL((verify_pick_kernel<T, E>), dim3(a.B), dim3(64), 0, st, a);
}

template <typename T>
void launch_verify(const VerifyArgs& a, int elems, hipStream_t st) {
  if (elems == 8)
    launch_verify<T, 8>(a, st);
  else
    launch_verify<T, 32>(a, st);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_verify_drafts_workspace(int64_t batch, int64_t drafts, int64_t vocab) {
  if (batch <= 0 || drafts <= 0 || vocab <= 0 || drafts > kVMaxDrafts || batch > 65535 ||
      vocab > INT32_MAX)
    return 0;
  const int elems = verify_elems(batch, vocab);
  const int64_t chunks = verify_chunks(vocab, elems), cells = batch * (2 * drafts + 1) * chunks;
  return 3 * up8(4 * cells) + 16 * batch * (verify_pieces(vocab, elems) + chunks) + 32 * batch;
}

extern "C" int32_t mi_verify_drafts(
    const void* target, const void* draft, const int64_t* drafted, const float* accept_u,
    const float* sample_u, const int64_t* draft_lens, int64_t* tokens, int64_t* accepted,
    void* workspace, int64_t workspace_bytes, int64_t batch, int64_t drafts, int64_t vocab,
    int64_t t_sb, int64_t t_ss, int64_t d_sb, int64_t d_ss, int64_t x_sb, int64_t x_ss,
    int64_t u_sb, int64_t u_ss, double temperature, int32_t dtype, void* stream) {
  if (dtype != MI_DTYPE_BF16 && dtype != MI_DTYPE_F16 && dtype != MI_DTYPE_F32) {
    set_last_error("verify_drafts: unknown dtype code");
    return MI_ERR_INVALID;
  }
  if (batch < 0 || drafts < 0 || vocab <= 0) {
    set_last_error("verify_drafts: invalid shape");
    return MI_ERR_INVALID;
  }
  if (!(temperature >= 0.0) || temperature > 1e6 || (temperature > 0.0 && temperature < 1e-3)) {
    set_last_error("verify_drafts: temperature must be 0 or between 1e-3 and 1e6");
    return MI_ERR_INVALID;
  }
  if (drafts < 1 || drafts > kVMaxDrafts || batch > 65535 || vocab > INT32_MAX ||
      batch * (2 * drafts + 1) > 65535) {
    set_last_error("verify_drafts: 1 to %d drafts, and batch * (2 * drafts + 1) <= 65535",
                   kVMaxDrafts);
    return MI_ERR_UNSUPPORTED;
  }
  if (batch == 0) return MI_OK;
  const bool greedy = temperature == 0.0;
  if (target == nullptr || drafted == nullptr || tokens == nullptr || accepted == nullptr ||
      workspace == nullptr || (!greedy && (accept_u == nullptr || sample_u == nullptr))) {
    set_last_error("verify_drafts: null pointer");
    return MI_ERR_INVALID;
  }
  if ((uintptr_t)workspace % 8 != 0 ||
      workspace_bytes < mi_verify_drafts_workspace(batch, drafts, vocab)) {
    set_last_error("verify_drafts: needs an 8-byte aligned workspace of %lld bytes",
                   (long long)mi_verify_drafts_workspace(batch, drafts, vocab));
    return MI_ERR_INVALID;
  }
  VerifyArgs a{};
  a.target = target;
  a.draft = greedy ? nullptr : draft;
  a.drafted = drafted; a.u = accept_u; a.r = sample_u; a.lens = draft_lens;
  a.tokens = tokens; a.accepted = accepted;
  a.B = (int32_t)batch; a.S = (int32_t)drafts; a.V = vocab;
  a.rows = (int32_t)(a.draft != nullptr ? 2 * drafts + 1 : drafts + 1);
  const int elems = verify_elems(batch, vocab);
  a.chunks = (int32_t)verify_chunks(vocab, elems);
  a.greedy = greedy;
  a.c = greedy ? 0.0 : 1.44269504088896340736 / temperature;
  const int64_t cells = batch * a.rows * a.chunks;
  char* w = static_cast<char*>(workspace);
  a.wsum = reinterpret_cast<double*>(w); w += 16 * batch * verify_pieces(vocab, elems);
  a.zsum = reinterpret_cast<double*>(w); w += 16 * batch * a.chunks;
  a.fin = reinterpret_cast<double*>(w); w += 32 * batch;
  a.sums = reinterpret_cast<float*>(w); w += up8(4 * cells);
  a.tops = reinterpret_cast<float*>(w); w += up8(4 * cells);
  a.args = reinterpret_cast<int32_t*>(w);
  a.t_sb = t_sb; a.t_ss = t_ss; a.d_sb = d_sb; a.d_ss = d_ss;
  a.x_sb = x_sb; a.x_ss = x_ss; a.u_sb = u_sb; a.u_ss = u_ss;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MI_DTYPE_BF16)
    launch_verify<bf16_t>(a, elems, st);
  else if (dtype == MI_DTYPE_F16)
    launch_verify<f16_t>(a, elems, st);
  else
    launch_verify<float>(a, elems, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_last_error("verify_drafts: launch failed: %s", hipGetErrorString(e));
    return (int32_t)e;
  }
  return MI_OK;
}
