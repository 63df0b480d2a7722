// Verification of drafted tokens against the target model's probabilities, from
// given uniform numbers, so that the tokens kept are distributed as if drawn
// from the target alone.
//
// p_n, q_n: the target's and the drafter's probabilities after node n, softmax(
// logits / T).  The walk starts at node 0 and takes nodes in order; a child i of
// the current node n, token x, is accepted with probability r(x) / q_n(x), where
// r starts as p_n and becomes norm(max(r - q_n, 0)) after each rejection.  All
// of those residuals are of one form, with one number c per node:
//   r = max(p - c q, 0) / S(c),   S(c) = sum_t max(p(t) - c q(t), 0),
// c = 0 (S = 1) at first, and r - q is proportional to p - (c + S(c)) q, so a
// rejection is c += S(c).  The test is u_i q(x) S(c) < p(x) - c q(x).  The token
// after the last accepted node is drawn from its r by inversion with u_0.
// Without a drafter's logits each token is a certain proposal: r is p without
// the tokens rejected so far, and the test is u_i (1 - their mass) < p(x).
//
// Sums and probabilities are held in 64 bits: a token's border in the
// cumulative sum over V tokens is off by V times a term's error, which in 32
// bits would exceed the width of unlikely tokens.
#include <float.h>

#include "hn_common.h"

namespace {

constexpr int kMaxNodes = 256;
constexpr int kThreads = 1024;
constexpr double kTiny = 0x1p-40;  // residual mass below which nothing is left

typedef __bf16 b16;

template <typename T>
__device__ __forceinline__ float logit(const T* p) {
  const float x = (float)*p;
  return x == x ? fminf(x, FLT_MAX) : -__builtin_inff();
}

struct Row {
  double m;   // largest logit
  double iz;  // 1 / sum exp((l - m) / T); 0: no token has a probability
};

template <typename T>
struct Walk {
  double it;  // 1 / T
  int V;
  double* red;  // [kThreads / 64]

  __device__ double sum(double x) {
    for (int off = 32; off; off >>= 1) x += __shfl_xor(x, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    double t = 0.;
    for (int w = 0; w < kThreads / 64; ++w) t += red[w];
    return t;
  }
  __device__ double largest(double x) {
    for (int off = 32; off; off >>= 1) x = fmax(x, __shfl_xor(x, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    double t = red[0];
    for (int w = 1; w < kThreads / 64; ++w) t = fmax(t, red[w]);
    return t;
  }
  __device__ Row row(const T* p) {
    double m = -__builtin_inf();
    for (int t = threadIdx.x; t < V; t += kThreads) m = fmax(m, (double)logit(p + t));
    m = largest(m);
    double s = 0.;
    if (m > -__builtin_inf())
      for (int t = threadIdx.x; t < V; t += kThreads) s += exp(((double)logit(p + t) - m) * it);
    s = sum(s);
    return Row{m, s > 0. ? 1. / s : 0.};
  }
  __device__ double prob(const T* p, const Row& r, int t) const {
    return r.iz > 0. ? exp(((double)logit(p + t) - r.m) * it) * r.iz : 0.;
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void verify_kernel(
    const T* __restrict__ logits, long sb, long ss, const T* __restrict__ draft, long db, long ds,
    const long* __restrict__ tokens, const int* __restrict__ up, int trees,
    const float* __restrict__ u, const float* __restrict__ temp, float temp0, int S, int V,
    int* __restrict__ path, int* __restrict__ count, long* __restrict__ token) {
  __shared__ double red[kThreads / 64];
  __shared__ int s_up[kMaxNodes];
  __shared__ long s_tok[kMaxNodes];
  __shared__ float s_u[kMaxNodes];
  __shared__ long gone[kMaxNodes];
  __shared__ double s_part[kThreads];
  __shared__ int s_pick;
  const int b = blockIdx.x, tid = threadIdx.x;
  for (int i = tid; i < S; i += kThreads) {
    s_up[i] = up[(trees > 1 ? (long)b * S : 0) + i];
    s_tok[i] = tokens[(long)b * S + i];
    s_u[i] = u[(long)b * S + i];
    path[(long)b * S + i] = i ? -1 : 0;
  }
  __syncthreads();
  const float tb = temp ? temp[b] : temp0;
  const bool greedy = !(tb > 0.f), soft = draft && !greedy;
  Walk<T> W = {greedy ? 1. : 1. / (double)tb, V, red};
  logits += b * sb;
  if (draft) draft += b * db;

  int cur = 0, n = 1, ngone = 0;
  double c = 0., mass = 1.;
  Row P = {}, Q = {};
  int top = -1;
  auto enter = [&]() {
    const T* p = logits + cur * ss;
    if (greedy) {
      double m = -__builtin_inf();
      for (int t = tid; t < V; t += kThreads) m = fmax(m, (double)logit(p + t));
      m = W.largest(m);
      int at = V;
      if (m > -__builtin_inf())
        for (int t = tid; t < V; t += kThreads)
          if ((double)logit(p + t) == m) at = at < t ? at : t;
      at = (int)-W.largest(-(double)at);
      top = at < V ? at : -1;
    } else {
      P = W.row(p);
      if (soft) Q = W.row(draft + cur * ds);
    }
    c = 0., mass = 1., ngone = 0;
  };
  auto left = [&](int t) -> double {
    const double p = W.prob(logits + cur * ss, P, t);
    return soft && c > 0. ? fmax(p - c * W.prob(draft + cur * ds, Q, t), 0.) : p;
  };
  enter();
  for (int i = 1; i < S; ++i) {
    if (s_up[i] != cur) continue;
    const long x = s_tok[i];
    const bool in = x >= 0 && x < V;
    bool take = false;
    if (greedy) {
      take = in && x == top;
    } else if (in && mass > kTiny) {
      const double px = W.prob(logits + cur * ss, P, (int)x);
      if (soft) {
        const double qx = W.prob(draft + cur * ds, Q, (int)x);
        take = (double)s_u[i] * qx * mass < px - c * qx;
      } else {
        bool was = false;
        for (int j = 0; j < ngone; ++j) was |= gone[j] == x;
        take = !was && (double)s_u[i] * mass < px;
        if (!take && !was) {
          mass -= px;
          __syncthreads();
          if (tid == 0) gone[ngone] = x;
          __syncthreads();
          ++ngone;
        }
      }
    }
    if (take) {
      cur = i;
      if (tid == 0) path[(long)b * S + n] = i;
      ++n;
      enter();
    } else if (soft && in && mass > kTiny) {
      c += mass;
      double s = 0.;
      for (int t = tid; t < V; t += kThreads) s += left(t);
      mass = W.sum(s);
    }
  }
  if (tid == 0) count[b] = n;
  if (greedy) {
    if (tid == 0) token[b] = top;
    return;
  }
  if (!(mass > kTiny)) c = 0., ngone = 0;  // nothing left: the target itself
  // inversion: a run of tokens per thread, then the run that holds the target
  const int per = (V + kThreads - 1) / kThreads, t0 = tid * per;
  const int t1 = t0 + per < V ? t0 + per : V;
  auto value = [&](int t) -> double {
    for (int j = 0; j < ngone; ++j)
      if (gone[j] == t) return 0.;
    return left(t);
  };
  double s = 0.;
  int last = -1;
  for (int t = t0; t < t1; ++t) {
    const double r = value(t);
    s += r;
    if (r > 0.) last = t;
  }
  s_part[tid] = s;
  if (tid == 0) s_pick = V;
  __syncthreads();
  double before = 0., all = 0.;
  for (int j = 0; j < kThreads; ++j) {
    if (j < tid) before += s_part[j];
    all += s_part[j];
  }
  last = (int)W.largest((double)last);
  const double target = (double)s_u[0] * all;
  for (int t = t0; t < t1; ++t) {
    const double r = value(t);
    before += r;
    if (r > 0. && before > target) {
      atomicMin(&s_pick, t);
      break;
    }
  }
  __syncthreads();
  if (tid == 0) token[b] = s_pick < V ? s_pick : last;
}

}  // namespace

// See include/hn_int4.h.
extern "C" long hn_verify_tree_workspace_bytes(long B, long S, long V, int soft) { return 0; }

// See include/hn_int4.h.
extern "C" int hn_verify_tree(const void* logits, long ld_b, long ld_s, const void* draft,
                              long ld_db, long ld_ds, int dtype, const long* tokens, const int* up,
                              long trees, const float* u, const float* temps, float temperature,
                              long B, long S, long V, int* path, int* count, long* token,
                              void* work, long work_bytes, void* stream) {
  const char* who = "hn_verify_tree";
  HN_ARG_CHECK(B >= 0 && S >= 1 && S <= kMaxNodes && V >= 1 && V < (1L << 30),
               "%s: need 1 <= nodes <= %d and 1 <= vocabulary < 2^30", who, kMaxNodes);
  HN_ARG_CHECK(trees == 1 || trees == B, "%s: need one tree or one per sequence", who);
  HN_ARG_CHECK(dtype >= 0 && dtype <= 2, "%s: dtype must be 0 (fp16), 1 (bf16) or 2 (fp32)", who);
  HN_ARG_CHECK(temps || temperature >= 0.f, "%s: temperature must not be negative", who);
  HN_ARG_CHECK((S == 1 || ld_s >= V) && (!draft || S == 1 || ld_ds >= V),
               "%s: row strides below the vocabulary", who);
  if (B == 0) return 0;
  HN_ARG_CHECK(logits && tokens && up && u && path && count && token, "%s: null operand", who);
  HN_ARG_CHECK(B < (1L << 31), "%s: too many sequences", who);
#define HN_VERIFY(T)                                                                            \
  hipLaunchKernelGGL(verify_kernel<T>, dim3((unsigned)B), dim3(kThreads), 0, (hipStream_t)stream, \
                     (const T*)logits, ld_b, ld_s, (const T*)draft, ld_db, ld_ds, tokens, up,   \
                     (int)trees, u, temps, temperature, (int)S, (int)V, path, count, token)
  if (dtype == 0)
    HN_VERIFY(h16);
  else if (dtype == 1)
    HN_VERIFY(b16);
  else
    HN_VERIFY(float);
#undef HN_VERIFY
  HN_LAUNCH_CHECK(who);
  return 0;
}
