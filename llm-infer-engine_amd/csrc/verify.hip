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
// sums of fp32 shares do not resolve.  Shares and sums are therefore fp64
// (exp2_f64: a polynomial of 2^f to 1e-12, 17 instructions an element; the vector
// units run fp64 at fp32's rate).
//
// Three launches: `stats` reads every row that may matter once (chunks of 8192
// logits, each in its block's registers: largest value, its index, sum of shares
// relative to it); `decide`, one block a (row, chunk), joins the stats, decides and
// sums w over its chunk; `pick`, one block a row, finds the chunk and in it the
// token.  T = 0 needs the first two only.
#include <algorithm>

#include "common.hpp"

namespace mi {

constexpr int kVChunk = 8192;      // logits of a block: 32 a thread
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
  double* sums;
  float* tops;
  int32_t* args;
  double* wsum;       // [B, chunks, 2]: sums of w and of p
  double* fin;        // [B, 4]: largest value and 1 / sum of row n, of the target and of the draft
  int64_t t_sb, t_ss, d_sb, d_ss, x_sb, x_ss, u_sb, u_ss;
  int64_t V;
  double c;           // log2(e) / T
  int32_t B, S, rows, chunks, greedy;
};

// 2^y for y <= 0 to 1e-12 of its value: y = k + f, |f| <= 1/2, and the series of
// e^(f ln 2) to the 10th power (the next term is below 3e-13).
__device__ inline double exp2_f64(double y) {
  y = fmax(y, -1100.0);            // 2^-1100 is 0
  const double k = __builtin_rint(y);
  const double t = (y - k) * 0.69314718055994530942;
  double p = 1.0 / 3628800.0;
  p = fma(p, t, 1.0 / 362880.0);
  p = fma(p, t, 1.0 / 40320.0);
  p = fma(p, t, 1.0 / 5040.0);
  p = fma(p, t, 1.0 / 720.0);
  p = fma(p, t, 1.0 / 120.0);
  p = fma(p, t, 1.0 / 24.0);
  p = fma(p, t, 1.0 / 6.0);
  p = fma(p, t, 0.5);
  p = fma(p, t, 1.0);
  p = fma(p, t, 1.0);
  return ldexp(p, (int)k);
}

__device__ inline float logit(float x) {
  return x != x ? -INFINITY : fminf(x, 3.402823466e38f);
}

// share of a logit in a row whose largest is m (0 in a row without mass)
__device__ inline double share(float x, float m, double c) {
  return m == -INFINITY ? 0.0 : exp2_f64(((double)x - (double)m) * c);
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

// The thread's 32 logits of a chunk: groups of 16 bytes aligned in memory, dealt to
// the threads in turn.  `first` + index is a logit's place in the row; places
// outside the chunk's [lo, hi) hold -inf.
template <typename T>
struct ChunkLogits {
  static constexpr int N = Chunk<T>::kN;       // logits of a group
  static constexpr int G = 32 / N;             // groups of a thread
  float x[32];
  int64_t base;                                // place of group 0's first logit (may be < lo)
  __device__ inline int64_t place(int g) const { return base + ((int64_t)g * 256 + threadIdx.x) * N; }
  __device__ inline void load(const T* row, int64_t lo, int64_t hi) {
    // the chunk starts at the group that holds lo
    const int mis = (int)(((uintptr_t)(row + lo) % 16) / sizeof(T));
    base = lo - mis;
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int64_t j = place(g);
      if (j >= lo && j + N <= hi) {
        Chunk<T>::unpack(load16(row + j), x + g * N);
#pragma unroll
        for (int e = 0; e < N; ++e) x[g * N + e] = logit(x[g * N + e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          x[g * N + e] = j + e >= lo && j + e < hi ? logit(Elem<T>::to_f32(row[j + e])) : -INFINITY;
      }
    }
  }
};

// A chunk holds 8192 - 8 places: with a group's misalignment it still fits the threads.
constexpr int64_t kVPlaces = kVChunk - 8;

template <typename T>
__global__ __launch_bounds__(256) void verify_stats_kernel(VerifyArgs a) {
  __shared__ float top_s[4];
  __shared__ int64_t at_s[4];
  __shared__ double sum_s[4];
  const int chunk = blockIdx.x, row = blockIdx.y % a.rows, b = blockIdx.y / a.rows;
  const int n = drafts_of(a, b);
  if (row <= a.S ? row > n : row - a.S - 1 >= n) return;   // no draft there
  const int64_t lo = chunk * kVPlaces;
  const int64_t hi = lo + kVPlaces < a.V ? lo + kVPlaces : a.V;
  ChunkLogits<T> c;
  c.load(row_of<T>(a, b, row), lo, hi);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 32; ++i) top = fmaxf(top, c.x[i]);
  // least place of the thread's largest logit: its places grow with i
  int64_t at = INT64_MAX;
#pragma unroll
  for (int i = 31; i >= 0; --i)
    if (c.x[i] == top) at = c.place(i / c.N) + i % c.N;
  if (top == -INFINITY) at = lo;
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
  double sum = 0.0;
  if (!a.greedy && top > -INFINITY) {
#pragma unroll
    for (int i = 0; i < 32; ++i) sum += exp2_f64(((double)c.x[i] - (double)top) * a.c);
#pragma unroll
    for (int m = 32; m; m >>= 1) sum += __shfl_xor(sum, m, 64);
  }
  if ((threadIdx.x & 63) == 0) sum_s[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    const int64_t i = (int64_t)blockIdx.y * a.chunks + chunk;
    a.tops[i] = top;
    a.args[i] = (int32_t)at;
    a.sums[i] = sum_s[0] + sum_s[1] + sum_s[2] + sum_s[3];
  }
}

// the sum of a double over the block's 4 waves, in every thread
__device__ inline double block_sum(double x, double* lds) {
#pragma unroll
  for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  return lds[0] + lds[1] + lds[2] + lds[3];
}

// w and p of one logit pair of row n
struct Weights {
  float mt, md;
  double zt, zd, c;
  bool refused, model;
  int64_t point;      // the drafted token of a refused draft without logits, else -1
  __device__ inline void get(float t, float d, int64_t j, double* w, double* p) const {
    *p = share(t, mt, c) * zt;
    double q = 0.0;
    if (refused) q = model ? share(d, md, c) * zd : (j == point ? 1.0 : 0.0);
    const double left = *p - q;
    *w = left > 0.0 ? left : 0.0;
  }
};

template <typename T>
__global__ __launch_bounds__(256) void verify_decide_kernel(VerifyArgs a) {
  __shared__ float top_s[2 * kVMaxDrafts + 1];
  __shared__ double inv_s[2 * kVMaxDrafts + 1];
  __shared__ int32_t arg_s[2 * kVMaxDrafts + 1];
  __shared__ int first_s;
  __shared__ double red[4];
  const int chunk = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int n = drafts_of(a, b);
  if (tid == 0) first_s = n;
  for (int row = tid; row < a.rows; row += 256) {
    if (row <= a.S ? row > n : row - a.S - 1 >= n) continue;
    const int64_t i = ((int64_t)b * a.rows + row) * a.chunks;
    float top = -INFINITY;
    int32_t at = 0;
    for (int c = 0; c < a.chunks; ++c) {
      const float t = a.tops[i + c];
      if (t > top) {
        top = t;
        at = a.args[i + c];
      }
    }
    double z = 0.0;
    if (!a.greedy)
      for (int c = 0; c < a.chunks; ++c) z += share(a.tops[i + c], top, a.c) * a.sums[i + c];
    top_s[row] = top;
    arg_s[row] = top == -INFINITY ? -1 : at;
    inv_s[row] = z > 0.0 ? 1.0 / z : 0.0;
  }
  __syncthreads();
  const bool model = a.draft != nullptr;
  if (tid < n) {
    const int64_t x = a.drafted[b * a.x_sb + tid * a.x_ss];
    bool ok = false;
    if (x >= 0 && x < a.V) {
      if (a.greedy) {
        ok = x == arg_s[tid];
      } else {
        const double p = share(logit(Elem<T>::to_f32(row_of<T>(a, b, tid)[x])), top_s[tid], a.c) *
                         inv_s[tid];
        double q = 1.0;
        if (model) {
          const int dr = a.S + 1 + tid;
          q = share(logit(Elem<T>::to_f32(row_of<T>(a, b, dr)[x])), top_s[dr], a.c) * inv_s[dr];
        }
        ok = (double)a.u[b * a.u_sb + tid * a.u_ss] * q < p;
      }
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
  Weights w;
  w.refused = k < n;
  w.model = model;
  w.mt = top_s[k];
  w.zt = inv_s[k];
  w.md = w.refused && model ? top_s[a.S + 1 + k] : -INFINITY;
  w.zd = w.refused && model ? inv_s[a.S + 1 + k] : 0.0;
  w.c = a.c;
  w.point = w.refused && !model ? a.drafted[b * a.x_sb + k * a.x_ss] : -1;
  if (chunk == 0 && tid == 0) {
    double* f = a.fin + 4 * (int64_t)b;
    f[0] = w.mt;
    f[1] = w.zt;
    f[2] = w.md;
    f[3] = w.zd;
  }
  const int64_t lo = chunk * kVPlaces;
  const int64_t hi = lo + kVPlaces < a.V ? lo + kVPlaces : a.V;
  const T* tr = row_of<T>(a, b, k);
  const T* dr = w.refused && model ? row_of<T>(a, b, a.S + 1 + k) : nullptr;
  double ws = 0.0, ps = 0.0;
  if (dr != nullptr && ((uintptr_t)(tr + lo) - (uintptr_t)(dr + lo)) % 16 != 0) {
    // rows of different alignment: one logit at a time
    for (int64_t j = lo + tid; j < hi; j += 256) {
      double wj, pj;
      w.get(logit(Elem<T>::to_f32(tr[j])), logit(Elem<T>::to_f32(dr[j])), j, &wj, &pj);
      ws += wj;
      ps += pj;
    }
  } else {
    ChunkLogits<T> ct, cd;
    ct.load(tr, lo, hi);
    if (dr != nullptr) cd.load(dr, lo, hi);
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      double wj, pj;
      w.get(ct.x[i], dr != nullptr ? cd.x[i] : -INFINITY, ct.place(i / ct.N) + i % ct.N, &wj, &pj);
      ws += wj;
      ps += pj;
    }
  }
  ws = block_sum(ws, red);
  ps = block_sum(ps, red);
  if (tid == 0) {
    a.wsum[2 * ((int64_t)b * a.chunks + chunk)] = ws;
    a.wsum[2 * ((int64_t)b * a.chunks + chunk) + 1] = ps;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a) {
  __shared__ double pre_s[256];
  __shared__ double below_s;
  __shared__ int chunk_s;
  __shared__ long long hit_s, last_s;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int n = drafts_of(a, b), k = (int)a.accepted[b];
  const double* sums = a.wsum + 2 * (int64_t)b * a.chunks;
  double total = 0.0, total_p = 0.0;
  for (int c = 0; c < a.chunks; ++c) {
    total += sums[2 * c];
    total_p += sums[2 * c + 1];
  }
  const bool use_w = total > 0.0;              // else p itself (also where nothing was refused: w is p)
  if (!use_w) total = total_p;
  const double goal = (double)a.r[b] * total;
  if (tid == 0) {
    // the chunk in which the sum passes the goal; the last one with mass, should rounding pass none
    double run = 0.0, below = 0.0;
    int at = -1;
    for (int c = 0; c < a.chunks; ++c) {
      const double x = sums[2 * c + (use_w ? 0 : 1)];
      if (x > 0.0) {
        at = c;
        below = run;
        if (run + x > goal) break;
      }
      run += x;
    }
    chunk_s = at;
    below_s = below;
    hit_s = INT64_MAX;
    last_s = -1;
  }
  __syncthreads();
  int64_t* out = a.tokens + (int64_t)b * (a.S + 1) + k;
  if (chunk_s < 0) {                           // a row without mass: no token
    if (tid == 0) *out = -1;
    return;
  }
  Weights w;
  const double* f = a.fin + 4 * (int64_t)b;
  w.refused = k < n;
  w.model = a.draft != nullptr;
  w.mt = (float)f[0];
  w.zt = f[1];
  w.md = (float)f[2];
  w.zd = f[3];
  w.c = a.c;
  w.point = w.refused && !w.model ? a.drafted[b * a.x_sb + k * a.x_ss] : -1;
  const T* tr = row_of<T>(a, b, k);
  const T* dr = w.refused && w.model ? row_of<T>(a, b, a.S + 1 + k) : nullptr;
  const int64_t lo = chunk_s * kVPlaces;
  const int64_t hi = lo + kVPlaces < a.V ? lo + kVPlaces : a.V;
  // 32 places in a row for each thread, their sum, the sums before them, then the place
  const int64_t j0 = lo + 32 * tid;
  double mine = 0.0;
  for (int e = 0; e < 32; ++e) {
    const int64_t j = j0 + e;
    if (j >= hi) break;
    double wj, pj;
    w.get(logit(Elem<T>::to_f32(tr[j])), dr != nullptr ? logit(Elem<T>::to_f32(dr[j])) : -INFINITY, j, &wj, &pj);
    mine += use_w ? wj : pj;
  }
  pre_s[tid] = mine;
  __syncthreads();
  for (int s = 1; s < 256; s <<= 1) {          // inclusive sums over the threads
    const double x = tid >= s ? pre_s[tid - s] : 0.0;
    __syncthreads();
    pre_s[tid] += x;
    __syncthreads();
  }
  double run = below_s + (tid > 0 ? pre_s[tid - 1] : 0.0);
  if (mine > 0.0) {
    const bool over = below_s + pre_s[tid] > goal;
    long long last = -1;
    for (int e = 0; e < 32; ++e) {
      const int64_t j = j0 + e;
      if (j >= hi) break;
      double wj, pj;
      w.get(logit(Elem<T>::to_f32(tr[j])), dr != nullptr ? logit(Elem<T>::to_f32(dr[j])) : -INFINITY, j, &wj, &pj);
      const double x = use_w ? wj : pj;
      run += x;
      if (x > 0.0) {
        last = j;
        if (over && run > goal) {
          atomicMin((unsigned long long*)&hit_s, (unsigned long long)j);
          break;
        }
      }
    }
    // (the sums of one place after the other may end a rounding below the thread's sum)
    if (over) atomicMin((unsigned long long*)&hit_s, (unsigned long long)last);
    atomicMax(&last_s, last);
  }
  __syncthreads();
  if (tid == 0) *out = hit_s != INT64_MAX ? hit_s : last_s;
}

namespace {

int64_t verify_chunks(int64_t vocab) { return (vocab + kVPlaces - 1) / kVPlaces; }
int64_t up8(int64_t bytes) { return (bytes + 7) / 8 * 8; }

template <typename T>
void launch_verify(const VerifyArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(verify_stats_kernel<T>, dim3(a.chunks, a.B * a.rows), dim3(256), 0, st, a);
  hipLaunchKernelGGL(verify_decide_kernel<T>, dim3(a.greedy ? 1 : a.chunks, a.B), dim3(256), 0, st, a);
  if (!a.greedy)
    hipLaunchKernelGGL(verify_pick_kernel<T>, dim3(a.B), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace mi

using namespace mi;

extern "C" int64_t mi_verify_drafts_workspace(int64_t batch, int64_t drafts, int64_t vocab) {
  if (batch <= 0 || drafts <= 0 || vocab <= 0 || drafts > kVMaxDrafts || batch > 65535 ||
      vocab > INT32_MAX)
    return 0;
  const int64_t chunks = verify_chunks(vocab), cells = batch * (2 * drafts + 1) * chunks;
  return 8 * cells + up8(4 * cells) + up8(4 * cells) + 16 * batch * chunks + 32 * batch;
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
  a.chunks = (int32_t)verify_chunks(vocab);
  a.greedy = greedy;
  a.c = greedy ? 0.0 : 1.44269504088896340736 / temperature;
  const int64_t cells = batch * a.rows * a.chunks;
  char* w = static_cast<char*>(workspace);
  a.sums = reinterpret_cast<double*>(w); w += 8 * cells;
  a.wsum = reinterpret_cast<double*>(w); w += 16 * batch * a.chunks;
  a.fin = reinterpret_cast<double*>(w); w += 32 * batch;
  a.tops = reinterpret_cast<float*>(w); w += up8(4 * cells);
  a.args = reinterpret_cast<int32_t*>(w);
  a.t_sb = t_sb; a.t_ss = t_ss; a.d_sb = d_sb; a.d_ss = d_ss;
  a.x_sb = x_sb; a.x_ss = x_ss; a.u_sb = u_sb; a.u_ss = u_ss;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == MI_DTYPE_BF16)
    launch_verify<bf16_t>(a, st);
  else if (dtype == MI_DTYPE_F16)
    launch_verify<f16_t>(a, st);
  else
    launch_verify<float>(a, st);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_last_error("verify_drafts: launch failed: %s", hipGetErrorString(e));
    return (int32_t)e;
  }
  return MI_OK;
}
