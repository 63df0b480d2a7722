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
//
// stats_kernel reads every row once, over the whole chip: per row and chunk of
// tokens the largest logit, its index and the sum of exponentials.  With a
// drafter's logits, first_kernel has S(1) of the nodes whose first child is
// rejected in the same way, and node_kernel what becomes of each node's children.
// walk_kernel, one workgroup per sequence, follows that, or tests certain
// proposals in LDS, and reads a row again only for the draw: one chunk.
//
// Times: 5 nodes over 32000 tokens, greedy, one sequence: stats 4.2 us, walk 3.4
// (latency of two launches).  8 trees of 61 nodes, 4 children each, over 32000,
// fp16: stats 22 us, first 16, node 41, walk 13.  32 chains of 6 over 128000, fp32:
// 48 (4.4 TB/s), 25, 6, 14.  Certain proposals, whole calls: the 8 trees 46 us, the 32
// chains 44 (their rows 20 at a copy's rate), 5 nodes of one sequence 23.  Of the 22 us half are the 26 million exponentials at
// 19 vector instructions each, the rest their rows' arrival; the 41 are three passes
// by one workgroup, one after the other since each needs the mass that the last one
// left.  With little gain there (47 to 44 us together, without the shorter passes):
// leaving out nodes that the walk cannot reach, the next block's loads under the
// arithmetic, four exponentials interleaved.
#include <float.h>

#include "hn_common.h"

namespace {

constexpr int kMaxNodes = 256;
constexpr double kTiny = 0x1p-40;  // residual mass below which nothing is left

typedef __bf16 b16;

// exp(d) for d <= 0 in 64 bits: 2^(k / 32) from a table (32 entries: 64 lanes
// read them without a bank conflict), the rest, at most ln 2 / 64, by four terms
// of its series: relative error 2e-12.  About a dozen instructions, so a row's sum
// costs no more than reading it.
constexpr double kLn2 = 0.693147180559945309417;
constexpr int kTab = 32;

__device__ __forceinline__ void fill_table(double* tab) {  // by a workgroup; a barrier follows
  if (threadIdx.x < kTab) {
    const double x = threadIdx.x * (kLn2 / kTab);
    double y = 1.;
#pragma unroll
    for (int i = 20; i > 0; --i) y = 1. + y * x * (1. / i);
    tab[threadIdx.x] = y;
  }
}

// k: kTab / (T ln 2); of (l - m) / T
__device__ __forceinline__ double exp_of(const double* tab, float l, double m, double k) {
  constexpr double a = kLn2 / kTab, magic = 0x1.8p52;
  // -40000 / 32 is past the smallest double: 0, as for -inf
  double x = ((double)l - m) * k;
  x = x > -40000. ? x : -40000.;
  const double t = x + magic;
  const int i = (int)__builtin_bit_cast(unsigned long long, t);
  const double r = x - (t - magic);
  const double y =
      1. + r * (a + r * (a * a / 2. + r * (a * a * a / 6. + r * (a * a * a * a / 24.))));
  return __builtin_ldexp(y * tab[i & (kTab - 1)], i >> 5);
}

// A NaN logit counts as -inf, +inf as the largest finite number.
__device__ __forceinline__ float sane(float x) {
  return fminf(fmaxf(x, -__builtin_inff()), FLT_MAX);
}

// 8 logits from any address, -inf past the end
template <typename T>
__device__ __forceinline__ void load8(float x[8], const T* p, int left) {
  typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  if (left >= 8) {
    const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = sane((float)v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < left ? sane((float)p[i]) : -__builtin_inff();
  }
}

// x of another lane by a data-parallel-primitive move, 0 where there is none
template <int CTL, int ROWS = 0xf>
__device__ __forceinline__ double moved(double x) {
  const unsigned long long w = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)w, CTL, ROWS, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(w >> 32), CTL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
// Sums of the lanes up to each, within rows of 16, then over the rows.
__device__ __forceinline__ double scan(double x) {
  x += moved<0x111>(x);  // row_shr:1, 2, 4, 8
  x += moved<0x112>(x);
  x += moved<0x114>(x);
  x += moved<0x118>(x);
  x += moved<0x142, 0xa>(x);  // row_bcast:15 into rows 1 and 3
  x += moved<0x143, 0xc>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ double lane_of(double x, int l) {
  const unsigned long long w = __builtin_bit_cast(unsigned long long, x);
  const unsigned lo = __builtin_amdgcn_readlane((int)w, l);
  const unsigned hi = __builtin_amdgcn_readlane((int)(w >> 32), l);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}

// What a chunk of a row comes to.
struct Part {
  float m;   // largest logit
  int at;    // its lowest index
  double s;  // sum of exp((l - m) / T)
};

// Chunks: a multiple of kBlock tokens, at most 64 of them.
constexpr int kBlock = 8192;
constexpr int kMaxChunks = 64;
struct Chunks {
  int n, size;
};
__host__ __device__ inline Chunks chunks_of(long V) {
  const long blocks = (V + kBlock - 1) / kBlock, per = (blocks + kMaxChunks - 1) / kMaxChunks;
  return Chunks{(int)((blocks + per - 1) / per), (int)(per * kBlock)};
}

struct Next;
struct Verify {
  const void *logits, *draft;
  long sb, ss, db, ds;
  const long* tokens;
  const int* up;
  const float *u, *temps;
  float temp;
  int trees, S, V;
  int* path;
  int* count;
  long* token;
  Part* part;     // [B][2][S][chunks]: the target's rows, the drafter's
  double* first;  // [B][S][chunks]: the last S(c) of a node whose first child is rejected, or -1
  Next* next;           // [B][S]
};

constexpr int kStat = 256;

// Grid (chunks, rows, B): the target's rows of the tree's nodes, then the
// drafter's rows of nodes that have children.
template <typename T>
__global__ __launch_bounds__(kStat) void stats_kernel(Verify A) {
  constexpr int kVec = kBlock / kStat / 8;  // vectors of 8 per thread and block
  __shared__ double tab[kTab], s_s[kStat / 64];
  __shared__ float s_m[kStat / 64];
  __shared__ int s_at[kStat / 64];
  const int b = blockIdx.z, tid = threadIdx.x, wave = tid >> 6;
  const bool dr = (int)blockIdx.y >= A.S;
  const int node = blockIdx.y - (dr ? A.S : 0);
  const int* up = A.up + (A.trees > 1 ? (long)b * A.S : 0);
  const float t = A.temps ? A.temps[b] : A.temp;
  const bool greedy = !(t > 0.f);
  fill_table(tab);
  const double k = greedy ? 0. : kTab / ((double)t * kLn2);
  const T* row = (const T*)(dr ? A.draft : A.logits) +
                 (dr ? b * A.db + node * A.ds : b * A.sb + node * A.ss);
  const Chunks C = chunks_of(A.V);
  const int t0 = blockIdx.x * C.size, t1 = t0 + C.size < A.V ? t0 + C.size : A.V;
  float x[kVec][8];
  auto load = [&](int o) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const int e = o + (j * kStat + tid) * 8;
      load8(x[j], row + e, e < t1 ? t1 - e : 0);
    }
  };
  if (!dr) load(t0);  // under the round trip of the checks
  if (dr && greedy) return;
  if (node && up[node] == -2) return;
  if (dr) {
    bool inner = false;
    for (int i = node + 1 + tid; i < A.S; i += kStat) inner |= up[i] == node;
    if (!__syncthreads_or(inner)) return;
  }
  Part P = {-__builtin_inff(), A.V, 0.};
  for (int o = t0; o < t1; o += kBlock) {
    if (dr || o > t0) load(o);
    float m = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kVec; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, x[j][i]);
    const float mine = m;
    for (int off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
    __syncthreads();  // also the table, and the last block's reads of s_*
    if ((tid & 63) == 0) s_m[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStat / 64; ++w) m = fmaxf(m, s_m[w]);
    int at = A.V;
    double s = 0.;
    if (greedy) {
      if (mine == m && m > -__builtin_inff())
#pragma unroll
        for (int j = kVec - 1; j >= 0; --j)
#pragma unroll
          for (int i = 7; i >= 0; --i)
            if (x[j][i] == m) at = o + (j * kStat + tid) * 8 + i;
      for (int off = 32; off; off >>= 1) {
        const int q = __shfl_xor(at, off, 64);
        at = q < at ? q : at;
      }
    } else if (m > -__builtin_inff()) {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) s += exp_of(tab, x[j][i], m, k);
      s = scan(s);
    }
    if ((tid & 63) == 63) s_at[wave] = at, s_s[wave] = s;
    __syncthreads();
    if (tid == 0) {
      s = 0.;
#pragma unroll
      for (int w = 0; w < kStat / 64; ++w) {
        s += s_s[w];
        at = s_at[w] < at ? s_at[w] : at;
      }
      if (m > P.m) {
        if (!greedy) P.s = P.s * exp_of(tab, P.m, m, k) + s;
        P.m = m, P.at = at;
      } else if (!greedy && m > -__builtin_inff()) {
        P.s += s * exp_of(tab, m, P.m, k);
      }
    }
  }
  if (tid == 0) A.part[(((long)b * 2 + dr) * A.S + node) * C.n + blockIdx.x] = P;
}

// A row's largest logit and 1 / its sum of exponentials (0: no finite logit), by a
// wave, a lane per chunk; every lane has them.
struct RowStat {
  float m;
  double z;
};
__device__ __forceinline__ RowStat row_stat(const Part* p, int chunks, const double* tab, double k) {
  const int lane = threadIdx.x & 63;
  Part P = {-__builtin_inff(), 0, 0.};
  if (lane < chunks) P = p[lane];
  float m = P.m;
  for (int off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
  const bool any = m > -__builtin_inff();
  const double s = lane_of(scan(any ? P.s * exp_of(tab, P.m, m, k) : 0.), 63);
  return RowStat{m, s > 0. ? 1. / s : 0.};
}
__device__ __forceinline__ double prob_of(const double* tab, const RowStat& r, float l, double k) {
  return r.z > 0. ? exp_of(tab, l, r.m, k) * r.z : 0.;
}

// max(p - c q, 0) of 8 tokens
template <typename T>
struct Rows {
  const T *p, *q;
  double pm, pz, qm, qz;  // largest logits, 1 / sums (c's factor in the drafter's)
  bool both;              // c > 0

  __device__ Rows(const T* p_, const T* q_, RowStat P, RowStat Q, double c)
      : p(p_), q(q_), pm(P.z > 0. ? P.m : 0.), pz(P.z), qm(Q.z > 0. ? Q.m : 0.), qz(c * Q.z),
        both(c > 0.) {}  // without a finite logit: exponents of -inf, sums of 0
  __device__ __forceinline__ double left(float x, float y, const double* tab, double k) const {
    const double d = exp_of(tab, x, pm, k) * pz - exp_of(tab, y, qm, k) * qz;
    return d > 0. ? d : 0.;
  }
  __device__ __forceinline__ void left8(double r[8], const double* tab, double k, int e,
                                        int end) const {
    float x[8], y[8];
    load8(x, p + e, end - e);
    if (both) load8(y, q + e, end - e);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = exp_of(tab, x[i], pm, k) * pz;
    if (both) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double d = r[i] - exp_of(tab, y[i], qm, k) * qz;
        r[i] = d > 0. ? d : 0.;
      }
    }
  }
};

// The mass that a node's first rejection leaves, S(1), by chunks over the whole
// chip: the walk needs it at each node whose first child is rejected, and most
// trees need little more.  (A node that the walk does not come to is summed for
// nothing.)  -1 where that child is accepted.  Grid (chunks, S - 1, B).
template <typename T>
__global__ __launch_bounds__(kStat) void first_kernel(Verify A) {
  __shared__ double tab[kTab], s_s[kStat / 64];
  __shared__ int s_child;
  __shared__ bool s_need;
  const int b = blockIdx.z, node = blockIdx.y, tid = threadIdx.x;
  const int* up = A.up + (A.trees > 1 ? (long)b * A.S : 0);
  const long* tok = A.tokens + (long)b * A.S;
  const float t = A.temps ? A.temps[b] : A.temp;
  if (!(t > 0.f)) return;
  if (tid == 0) s_child = A.S;
  fill_table(tab);
  __syncthreads();
  for (int i = node + 1 + tid; i < A.S; i += kStat)
    if (up[i] == node && tok[i] >= 0 && tok[i] < A.V) {
      atomicMin(&s_child, i);
      break;
    }
  __syncthreads();
  const int child = s_child;
  if (child == A.S) return;
  const double k = kTab / ((double)t * kLn2);
  const Chunks C = chunks_of(A.V);
  const T* p = (const T*)A.logits + b * A.sb + node * A.ss;
  const T* q = (const T*)A.draft + b * A.db + node * A.ds;
  const RowStat P = row_stat(A.part + (((long)b * 2) * A.S + node) * C.n, C.n, tab, k);
  const RowStat Q = row_stat(A.part + (((long)b * 2 + 1) * A.S + node) * C.n, C.n, tab, k);
  if (tid == 0) {
    const double px = prob_of(tab, P, sane((float)p[tok[child]]), k);
    const double qx = prob_of(tab, Q, sane((float)q[tok[child]]), k);
    s_need = !((double)A.u[(long)b * A.S + child] * qx < px);
    if (!s_need) A.first[((long)b * A.S + node) * C.n + blockIdx.x] = -1.;
  }
  __syncthreads();
  if (!s_need) return;
  const Rows<T> R(p, q, P, Q, 1.);
  const int t0 = blockIdx.x * C.size, t1 = t0 + C.size < A.V ? t0 + C.size : A.V;
  double s = 0.;
  for (int e = t0 + tid * 8; e < t1; e += kStat * 8) {
    double r[8];
    R.left8(r, tab, k, e, t1);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += r[i];
  }
  s = scan(s);
  if ((tid & 63) == 63) s_s[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.;
#pragma unroll
    for (int w = 0; w < kStat / 64; ++w) s += s_s[w];
    A.first[((long)b * A.S + node) * C.n + blockIdx.x] = s;
  }
}

constexpr int kWalk = 1024, kWaves = kWalk / 64;

// A chunk's mass, each wave's part of it into sum[ch], by a workgroup of kWalk.
template <typename F>
__device__ __forceinline__ void sum_chunk(F left8, const Chunks& C, int V, int ch,
                                          double (*sum)[kWaves]) {
  const int t0 = ch * C.size, t1 = t0 + C.size < V ? t0 + C.size : V, tid = threadIdx.x;
  double s = 0.;
  for (int e = t0 + tid * 8; e < t1; e += kWalk * 8) {
    double r[8];
    left8(r, e, t1);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += r[i];
  }
  s = scan(s);
  if ((tid & 63) == 63) sum[ch][tid >> 6] = s;
}

// Where the walk goes from a node, with a drafter's logits: a workgroup per node,
// since a node's tests start at c = 0 whatever came before, so all nodes' further
// rejections (a pass over both rows each) run side by side.
struct Next {
  int node;        // the accepted child, or -1
  double c, mass;  // else the residual's c and S(c); its chunks' masses are in first
};

// The tokens that a pass leaves mass, as c only grows the only ones that the next can:
// the logits of those that a wave came by, in its order, and where its chunks end.  A
// third of 32000 tokens or less in trees of 4 children each, whose nodes took 47 us
// with each pass over whole rows and 41 with the passes after the first over these.
// Where they do not fit, the next pass reads the rows again.
template <typename T>
struct Kept {
  static constexpr int kMost = 2048 / sizeof(T);  // 64 KB: two workgroups per CU
  struct Two {
    T p, q;
  } of[kWaves][kMost];
  unsigned short end[kMaxChunks][kWaves];
};

template <typename T>
__global__ __launch_bounds__(kWalk) void node_kernel(Verify A) {
  __shared__ double tab[kTab];
  __shared__ RowStat s_stat[2];
  __shared__ double s_px[kMaxNodes], s_qx[kMaxNodes];
  __shared__ float s_u[kMaxNodes];
  __shared__ bool s_kid[kMaxNodes];  // a child whose token is in the vocabulary
  __shared__ double s_sum[kMaxChunks][kWaves];
  __shared__ Kept<T> s_kept;
  __shared__ int s_last;
  const int b = blockIdx.y, node = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), S = A.S, V = A.V;
  const float t = A.temps ? A.temps[b] : A.temp;
  if (!(t > 0.f)) return;
  const int* up = A.up + (A.trees > 1 ? (long)b * S : 0);
  const T* p = (const T*)A.logits + b * A.sb + node * A.ss;
  const T* q = (const T*)A.draft + b * A.db + node * A.ds;
  float lp = 0.f, lq = 0.f;
  bool kid = false;
  if (tid > node && tid < S && up[tid] == node) {
    const long x = A.tokens[(long)b * S + tid];
    kid = x >= 0 && x < V;
    if (kid) lp = sane((float)p[x]), lq = sane((float)q[x]), s_u[tid] = A.u[(long)b * S + tid];
  }
  if (tid < S) s_kid[tid] = kid;
  if (tid == 0) s_last = 0;
  fill_table(tab);
  Next N = {-1, 0., 1.};
  if (__syncthreads_or(kid)) {
    if (kid) atomicMax(&s_last, tid);
    const double k = kTab / ((double)t * kLn2);
    const Chunks C = chunks_of(V);
    if (tid < 128) {
      const RowStat R =
          row_stat(A.part + (((long)b * 2 + (tid >> 6)) * S + node) * C.n, C.n, tab, k);
      if (lane == 0) s_stat[tid >> 6] = R;
    }
    __syncthreads();
    if (kid) {
      s_px[tid] = prob_of(tab, s_stat[0], lp, k);
      s_qx[tid] = prob_of(tab, s_stat[1], lq, k);
    }
    __syncthreads();
    double* first = A.first + ((long)b * S + node) * C.n;
    const double left = lane < C.n ? first[lane] : 0.;  // by the first child's rejection
    bool again = false, kept = false;
    for (int i = node + 1; i < S && N.mass > kTiny; ++i) {
      if (!s_kid[i]) continue;
      if (N.c > 0. ? (double)s_u[i] * s_qx[i] * N.mass < s_px[i] - N.c * s_qx[i]
                   : lane_of(left, 0) < 0.) {
        N.node = i;
        break;
      }
      double s = 0.;
      if (N.c > 0.) {
        N.c += N.mass, again = true;
        const Rows<T> R(p, q, s_stat[0], s_stat[1], N.c);
        __syncthreads();  // the last sums are read
        if (kept) {
          for (int ch = 0, j = 0; ch < C.n; ++ch) {
            const int end = s_kept.end[ch][wave];
            double part = 0.;
            for (int e = j + lane; e < end; e += 64) {
              const auto w = s_kept.of[wave][e];
              part += R.left(sane((float)w.p), sane((float)w.q), tab, k);
            }
            part = scan(part);
            if (lane == 63) s_sum[ch][wave] = part;
            j = end;
          }
          __syncthreads();
        } else if (i < s_last) {  // there may be another pass
          int len = 0;
          for (int ch = 0; ch < C.n; ++ch) {
            const int t0 = ch * C.size, t1 = t0 + C.size < V ? t0 + C.size : V;
            double part = 0.;
            for (int o = t0; o < t1; o += kBlock) {
              float x[8], y[8];
              const int at = o + tid * 8;
              load8(x, p + at, t1 - at);
              load8(y, q + at, t1 - at);
              double r[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) r[e] = R.left(x[e], y[e], tab, k);
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                part += r[e];
                const unsigned long long some = __ballot(r[e] > 0.);
                const int to = len + __builtin_amdgcn_mbcnt_hi(
                                         some >> 32, __builtin_amdgcn_mbcnt_lo((unsigned)some, 0));
                if (r[e] > 0. && to < Kept<T>::kMost) s_kept.of[wave][to] = {(T)x[e], (T)y[e]};
                len += __popcll(some);
              }
            }
            part = scan(part);
            if (lane == 63) s_sum[ch][wave] = part;
            if (lane == 0) s_kept.end[ch][wave] = len < Kept<T>::kMost ? len : Kept<T>::kMost;
          }
          kept = !__syncthreads_or(len > Kept<T>::kMost);
        } else {
          for (int ch = 0; ch < C.n; ++ch)
            sum_chunk([&](double r[8], int e, int end) { R.left8(r, tab, k, e, end); }, C, V, ch,
                      s_sum);
          __syncthreads();
        }
        for (int j = lane; j < C.n * kWaves; j += 64) s += s_sum[j / kWaves][j % kWaves];
      } else {
        N.c = 1., s = left;
      }
      N.mass = lane_of(scan(s), 63);
    }
    if (N.node < 0 && again && tid < C.n) {
      double s = 0.;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += s_sum[tid][w];
      first[tid] = s;
    }
  }
  if (tid == 0) A.next[(long)b * S + node] = N;
}

// The walk from node 0, one workgroup per sequence, and the draw.
template <typename T>
__global__ __launch_bounds__(kWalk) void walk_kernel(Verify A) {
  __shared__ double tab[kTab];
  __shared__ RowStat s_stat[2];
  __shared__ int s_up[kMaxNodes], s_tok[kMaxNodes], s_top[kMaxNodes], s_gone[kMaxNodes];
  __shared__ float s_u[kMaxNodes];
  __shared__ double s_p[kMaxNodes], s_mass[kMaxNodes];  // p of a node's token; or Next's c, mass
  __shared__ double s_sum[kMaxChunks][kWaves], s_tot[kMaxChunks], s_scan[kWaves];
  __shared__ int s_pick, s_last;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int S = A.S, V = A.V;
  const Chunks C = chunks_of(V);
  const float tb = A.temps ? A.temps[b] : A.temp;
  const bool greedy = !(tb > 0.f), soft = A.draft && !greedy;
  const double k = greedy ? 0. : kTab / ((double)tb * kLn2);
  const T* lg = (const T*)A.logits + b * A.sb;
  const T* dl = soft ? (const T*)A.draft + b * A.db : nullptr;
  const Part* part = A.part + (long)b * 2 * S * C.n;  // the target's rows
  if (tid < S) {
    const int up = tid ? A.up[(A.trees > 1 ? (long)b * S : 0) + tid] : -1;
    if (soft) {
      const Next N = A.next[(long)b * S + tid];
      s_up[tid] = N.node, s_p[tid] = N.c, s_mass[tid] = N.mass;
    } else {
      const long x = A.tokens[(long)b * S + tid];
      s_up[tid] = up;
      s_tok[tid] = x >= 0 && x < V ? (int)x : -1;
    }
    s_u[tid] = A.u[(long)b * S + tid];
    A.path[(long)b * S + tid] = tid ? -1 : 0;
  }
  fill_table(tab);
  __syncthreads();

  int cur = 0, n = 1, ngone = 0;
  double c = 0., mass = 1.;
  auto accept = [&](int i) {
    cur = i;
    if (tid == 0) A.path[(long)b * S + n] = i;
    ++n;
  };
  if (soft) {
    for (int i = s_up[0]; i > cur; i = s_up[cur]) accept(i);
    c = s_p[cur], mass = s_mass[cur];
  } else {
    // a wave per row: its largest logit's index, or 1 / its sum and, of the row's
    // children, their tokens' probabilities
    for (int node = wave; node < S; node += kWaves) {
      if (s_up[node] == -2) continue;
      const Part* pr = part + (long)node * C.n;
      if (greedy) {
        Part P = {-__builtin_inff(), V, 0.};
        if (lane < C.n) P = pr[lane];
        float m = P.m;
        for (int off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
        int at = P.m == m && m > -__builtin_inff() ? P.at : V;
        for (int off = 32; off; off >>= 1) {
          const int q = __shfl_xor(at, off, 64);
          at = q < at ? q : at;
        }
        if (lane == 0) s_top[node] = at < V ? at : -1;
      } else {
        const RowStat R = row_stat(pr, C.n, tab, k);
        for (int i = node + 1 + lane; i < S; i += 64)
          if (s_up[i] == node && s_tok[i] >= 0)
            s_p[i] = prob_of(tab, R, sane((float)lg[node * A.ss + s_tok[i]]), k);
      }
    }
    __syncthreads();
    for (int i = 1; i < S; ++i) {
      if (s_up[i] != cur || s_tok[i] < 0) continue;
      const int x = s_tok[i];
      if (greedy) {
        if (x == s_top[cur]) accept(i);
        continue;
      }
      if (!(mass > kTiny)) continue;
      bool was = false;
      for (int j = 0; j < ngone; ++j) was |= s_gone[j] == x;
      if (was) continue;
      if ((double)s_u[i] * mass < s_p[i]) {
        accept(i), mass = 1., ngone = 0;
      } else {
        mass -= s_p[i];
        __syncthreads();
        if (tid == 0) s_gone[ngone] = x;
        __syncthreads();
        ++ngone;
      }
    }
  }
  if (tid == 0) A.count[b] = n;
  if (greedy) {
    if (tid == 0) A.token[b] = s_top[cur];
    return;
  }
  if (!(mass > kTiny)) c = 0., ngone = 0;  // nothing left: the target itself

  // The draw: the chunk that the target falls into, then the token.  The chunks'
  // masses are those of the last rejection, or the row's own sums, where a token
  // is gone anew.
  if (tid < (soft ? 128 : 64)) {
    const Part* pr = part + ((long)(tid >> 6) * S + cur) * C.n;
    const RowStat R = row_stat(pr, C.n, tab, k);
    if (lane == 0) s_stat[tid >> 6] = R;
    if (c == 0. && tid < C.n) {
      const Part P = pr[tid];
      s_tot[tid] = P.m > -__builtin_inff() ? P.s * prob_of(tab, R, P.m, k) : 0.;
    }
  } else if (c > 0. && wave == kWaves - 1 && lane < C.n) {
    s_tot[lane] = A.first[((long)b * S + cur) * C.n + lane];
  }
  __syncthreads();
  const Rows<T> R(lg + cur * A.ss, soft ? dl + cur * A.ds : nullptr, s_stat[0],
                  soft ? s_stat[1] : RowStat{0.f, 0.}, c);
  // 8 tokens of the residual, less those gone
  auto left8 = [&](double r[8], int e, int end) {
    R.left8(r, tab, k, e, end);
    for (int j = 0; j < ngone; ++j) {
      const int g = s_gone[j] - e;
      if (g >= 0 && g < 8)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i == g) r[i] = 0.;
    }
  };
  for (int j = 0; j < ngone; ++j) {
    const int ch = s_gone[j] / C.size;
    bool done = false;
    for (int q = 0; q < j; ++q) done |= s_gone[q] / C.size == ch;
    if (!done) sum_chunk(left8, C, V, ch, s_sum);
  }
  if (tid == 0) s_pick = V, s_last = -1;
  __syncthreads();
  if (ngone) {
    if (tid < ngone) {
      double s = 0.;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += s_sum[s_gone[tid] / C.size][w];
      s_tot[s_gone[tid] / C.size] = s;  // the same value from every token of the chunk
    }
    __syncthreads();
  }
  // a lane per chunk
  const double tot = lane < C.n ? s_tot[lane] : 0., cum = scan(tot);
  const double target = (double)s_u[0] * lane_of(cum, 63);
  const unsigned long long some = __ballot(tot > 0.), over = __ballot(tot > 0. && cum > target);
  if (!some) {  // no logit is finite
    if (tid == 0) A.token[b] = -1;
    return;
  }
  // the last that has any, if none exceeds the target
  const int pick = over ? __builtin_ctzll(over) : 63 - __builtin_clzll(some);
  double before = lane_of(cum, pick) - lane_of(tot, pick);
  const int t0 = pick * C.size, t1 = t0 + C.size < V ? t0 + C.size : V;
  for (int o = t0; o < t1; o += kBlock) {
    const int e = o + tid * 8;
    double r[8], sum = 0.;
    if (e < t1)
      left8(r, e, t1);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = 0.;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += r[i];
    double run = scan(sum);
    if (lane == 63) s_scan[wave] = run;
    __syncthreads();
    double base = before, total = before;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) base += s_scan[w];
      total += s_scan[w];
    }
    run = base + run - sum;
    int hit = V, last = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      run += r[i];
      if (r[i] > 0.) {
        last = e + i;
        if (hit == V && run > target) hit = e + i;
      }
    }
    if (hit < V) atomicMin(&s_pick, hit);
    if (last >= 0) atomicMax(&s_last, last);
    before = total;
    __syncthreads();
    if (s_pick < V) break;
  }
  if (tid == 0) A.token[b] = s_pick < V ? s_pick : s_last;
}

}  // namespace

// See include/hn_int4.h.
extern "C" long hn_verify_tree_workspace_bytes(long B, long S, long V) {
  if (B <= 0 || S <= 0 || V <= 0) return 0;
  return B * S * (chunks_of(V).n * (long)(2 * sizeof(Part) + sizeof(double)) + sizeof(Next));
}

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
  HN_ARG_CHECK(B <= 65535, "%s: at most 65535 sequences", who);
  const long need = hn_verify_tree_workspace_bytes(B, S, V);
  HN_ARG_CHECK(work && ((uintptr_t)work & 15) == 0 && work_bytes >= need,
               "%s: needs a 16-byte aligned workspace of %ld bytes (got %ld)", who, need,
               work_bytes);
  const bool soft = draft && (temps || temperature > 0.f);
  Part* parts = (Part*)work;
  double* first = (double*)(parts + B * 2 * S * chunks_of(V).n);
  const Verify A = {logits, draft, ld_b,  ld_s,   ld_db,  ld_ds,  tokens, up,
                    u,      temps, temperature, (int)trees, (int)S, (int)V, path, count,
                    token,  parts, first, (Next*)(first + B * S * chunks_of(V).n)};
  const dim3 grid((unsigned)chunks_of(V).n, (unsigned)(soft ? 2 * S : S), (unsigned)B);
  const dim3 nodes((unsigned)chunks_of(V).n, (unsigned)(S - 1), (unsigned)B);
  const dim3 per_node((unsigned)S, (unsigned)B);
  hipStream_t st = (hipStream_t)stream;
#define HN_VERIFY(T)                                                            \
  do {                                                                          \
    hipLaunchKernelGGL(stats_kernel<T>, grid, dim3(kStat), 0, st, A);           \
    HN_LAUNCH_CHECK(who);                                                       \
    if (soft && S > 1) {                                                        \
      hipLaunchKernelGGL(first_kernel<T>, nodes, dim3(kStat), 0, st, A);        \
      HN_LAUNCH_CHECK(who);                                                     \
    }                                                                           \
    if (soft) {                                                                 \
      hipLaunchKernelGGL(node_kernel<T>, per_node, dim3(kWalk), 0, st, A);      \
      HN_LAUNCH_CHECK(who);                                                     \
    }                                                                           \
    hipLaunchKernelGGL(walk_kernel<T>, dim3((unsigned)B), dim3(kWalk), 0, st, A); \
  } while (0)
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
