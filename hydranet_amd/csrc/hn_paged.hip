// A paged KV cache: the append of a step's keys and values with the position
// rotation of its queries and keys, and the attention over the pages.
//
// A page holds `page` positions of every KV head: keys [page id][kv head][slot][hd],
// values [page id][kv head][slot / 8][hd][8].  Row b of the table names the pages of
// sequence b in order.  A sequence with C = lens[b] >= 0 cached positions adds rows
// starts[b] to starts[b + 1] of the step (one row, b, without starts) at positions C on;
// a row sees the positions up to its own.
#include "../../include/hn_int4.h"
#include "hn_lds_dma.h"
#include "hn_paged.h"

namespace {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

template <class T>
struct Vec;
template <>
struct Vec<h16> {
  typedef half8_t t;
  static constexpr uint32_t inf = 0x7c00u;
  static constexpr float less = 1.f;  // a second walk's probabilities, to a first's
  static __device__ __forceinline__ float4v mfma(t a, t b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Vec<b16> {
  typedef bf8 t;
  static constexpr uint32_t inf = 0x7f80u;
  static constexpr float less = 0x1p-40f;
  static __device__ __forceinline__ float4v mfma(t a, t b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

// ---------------------------------------------------------------------------
// The append.  Bytes are all there is: projections read, queries and pages written, 55 to 57
// us for prompts of 8928 tokens, 32 heads over 8 of 128 (224 MB, 3.9 to 4.1 TB/s; a large copy
// moves 5.2), 4.9 us for 64 single tokens, where the latency of lengths, tables and angles
// after each other counts.
//
// One thread per element, grid (T, nh + 2 nkv): rows and rotated parts of any alignment (the
// prompts 283 us, 64 single tokens 5.0).
template <class T>
__global__ __launch_bounds__(256) void append_kernel(Step P, const T* __restrict__ qkv, long ld,
                                                     const float* __restrict__ cos_t,
                                                     const float* __restrict__ sin_t, long rows,
                                                     int rd, int pairs, int nh, int hd,
                                                     T* __restrict__ q_out, T* __restrict__ k,
                                                     T* __restrict__ v) {
  const int t = blockIdx.x, head = blockIdx.y, d = threadIdx.x;
  const Row r = row_near(P, t);
  if (r.b < 0) {
    if (head < nh) q_out[((long)t * nh + head) * hd + d] = (T)0.f;
    return;
  }
  long pg = -1;
  const bool in = r.pos >= 0 && r.pos < rows && (pg = page_of(P, r.b, r.pos)) >= 0;
  const int slot = (int)(r.pos & (P.page - 1));
  const T* x = qkv + (long)t * ld + (long)head * hd;
  if (head >= nh + P.nkv) {
    const long at = (pg * P.nkv + head - nh - P.nkv) * P.page;
    if (in) v[(at + (slot & ~7)) * hd + d * 8 + (slot & 7)] = x[d];
    return;
  }
  float y = r.pos < 0 ? 0.f : __builtin_nanf("");
  if (in) {
    y = (float)x[d];
    if (d < rd) {
      const int other = pairs ? d ^ 1 : d < rd / 2 ? d + rd / 2 : d - rd / 2;
      const int a = pairs ? d >> 1 : d < rd / 2 ? d : d - rd / 2;
      const float z = (float)x[other];
      y = y * cos_t[r.pos * (rd / 2) + a] + (other > d ? -z : z) * sin_t[r.pos * (rd / 2) + a];
    }
  }
  if (head < nh) q_out[((long)t * nh + head) * hd + d] = (T)y;
  else if (in) k[((pg * P.nkv + head - nh) * P.page + slot) * hd + d] = (T)y;
}

// 16 bytes; those of many rows past the caches, which keep the queries and pages instead
// (the prompts 57 -> 54 us).
template <bool MANY, class T>
__device__ __forceinline__ typename Vec<T>::t once(const T* p) {
  const auto* v = reinterpret_cast<const typename Vec<T>::t*>(p);
  if constexpr (MANY) return __builtin_nontemporal_load(v);
  return *v;
}

// The same by 16-byte vectors.  Queries and keys: a thread has 16 elements of a head at a
// time, the two vectors of 8 pairs (or of 16 dimensions that stay), so their 8 angles stay
// in registers over its NI heads; HD / 16 threads a head, `across` heads of a token side by
// side.  Values: a thread has 8 dimensions of the new rows among 8 slots of a page, which
// are 128 consecutive bytes; it writes them whole where all 8 are new, else its rows' 2
// bytes each.
template <class T, int HD, int NI>
__global__ __launch_bounds__(256) void append_rows_kernel(
    Step P, const T* __restrict__ qkv, long ld, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, long rows, int rd, int pairs, int nh, int across, int qy,
    int qk, T* __restrict__ q_out, T* __restrict__ kc, T* __restrict__ vc) {
  typedef typename Vec<T>::t V8;
  constexpr int kUnits = HD / 16;
  const int tid = threadIdx.x;
  if ((int)blockIdx.x < qk) {
    const int u = tid % kUnits, slot = tid / kUnits;
    const int t = (blockIdx.x / qy) * (256 / kUnits / across) + slot / across;
    const int h0 = (blockIdx.x % qy) * across * NI + slot % across;
    const bool there = t < P.T;
    // where the 16 elements lie, and the first of their angles
    const bool turn = 16 * u < rd;
    const int lo = !turn || pairs ? 16 * u : 8 * u;
    const int hi = !turn || pairs ? lo + 8 : lo + rd / 2;
    const T* src = qkv + (long)(there ? t : 0) * ld;
    V8 x[NI], y[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int h = min(h0 + i * across, nh + P.nkv - 1);
      x[i] = once<NI == 4>(src + (long)h * HD + lo);
      y[i] = once<NI == 4>(src + (long)h * HD + hi);
    }
    const Row r = row_near(P, there ? t : P.T - 1);
    if (!there) return;
    const long pg = r.b >= 0 && r.pos >= 0 && r.pos < rows ? page_of(P, r.b, r.pos) : -1;
    if (pg >= 0 && turn) {
      float4v c[2], s[2];
      const long at = r.pos * (rd / 2) + 8 * u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        c[j] = *reinterpret_cast<const float4v*>(cos_t + at + 4 * j);
        s[j] = *reinterpret_cast<const float4v*>(sin_t + at + 4 * j);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const V8 a = x[i], b = y[i];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // pair j: elements 2 j and 2 j + 1 of both vectors, or j of each
          const float f = (float)(pairs ? (j < 4 ? a[2 * j] : b[(2 * j) & 7]) : a[j]);
          const float z = (float)(pairs ? (j < 4 ? a[(2 * j + 1) & 7] : b[(2 * j + 1) & 7]) : b[j]);
          const float cj = c[j >> 2][j & 3], sj = s[j >> 2][j & 3];
          const T f2 = (T)(f * cj - z * sj), z2 = (T)(z * cj + f * sj);
          if (!pairs) x[i][j] = f2, y[i][j] = z2;
          else if (j < 4) x[i][(2 * j) & 7] = f2, x[i][(2 * j + 1) & 7] = z2;
          else y[i][(2 * j) & 7] = f2, y[i][(2 * j + 1) & 7] = z2;
        }
      }
    }
    const T none = (T)(r.pos < 0 ? 0.f : __builtin_nanf(""));
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int h = h0 + i * across;
      if (h >= nh + P.nkv || (h >= nh && pg < 0)) continue;
      if (pg < 0)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[i][j] = y[i][j] = none;
      T* dst = h < nh ? q_out + ((long)t * nh + h) * HD
                      : kc + ((pg * P.nkv + h - nh) * P.page + (r.pos & (P.page - 1))) * HD;
      *reinterpret_cast<V8*>(dst + lo) = x[i];
      *reinterpret_cast<V8*>(dst + hi) = y[i];
    }
    return;
  }
  // The rows that share 8 slots are the first one's (of the run, or at the first slot); a
  // thread looks for those among `step` rows.
  const int cols = P.nkv * (HD / 8), step = P.starts ? 8 : 1;
  const long id = (long)(blockIdx.x - qk) * 256 + tid;
  const int g = (int)(id / cols), c = (int)(id - (long)g * cols) * 8;
  const long t0 = (long)g * step;
  Row r = row_near(P, (int)min(t0, (long)P.T - 1));
  int t = (int)t0;
  if (t0 >= P.T) return;
  const int end = min(t + step, P.T);
  const T* src = qkv + (long)(nh + P.nkv) * HD + c;
  while (t < end) {
    // (rows before the first sequence: r.b -1; behind the last: nothing follows)
    if (r.b < 0) {
      if (t >= P.starts[0]) return;
      t = P.starts[0];
      if (t >= end) return;
      r = row_from(P, t, 0);
      continue;
    }
    const int first = P.starts ? P.starts[r.b] : t, stop = P.starts ? min(P.starts[r.b + 1], P.T) : t + 1;
    int n = stop - t;  // rows to go on by
    if (r.pos >= 0) {
      const int in = (int)(r.pos & 7);
      n = min(n, 8 - in);
      const long pg = r.pos < rows && (in == 0 || t == first) ? page_of(P, r.b, r.pos) : -1;
      if (pg >= 0) {
        const int m = (int)min((long)n, rows - r.pos);
        const int slot = (int)(r.pos & (P.page - 1));
        T* dst = vc + ((pg * P.nkv + c / HD) * P.page + (slot & ~7)) * HD + (c % HD) * 8;
        V8 x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[j] = once<NI == 4>(src + (long)(t + min(j, m - 1)) * ld);
        if (m == 8) {
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            V8 y;
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = x[j][d];
            *reinterpret_cast<V8*>(dst + 8 * d) = y;
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (j < m)
#pragma unroll
              for (int d = 0; d < 8; ++d) dst[8 * d + in + j] = x[j][d];
        }
      }
    }
    t += n;
    if (t < end) r = row_from(P, t, r.b);
  }
}

// ---------------------------------------------------------------------------
// Attention.  One pass over a sequence's pages with a running maximum and sum, for the
// rows of one (sequence, KV head), a row being a (new token, query head of the group)
// pair.  A wave takes 32 positions at a time:
//   S^T = K Q^T    v_mfma_f32_16x16x32, A = K, B = Q, two blocks of 16 positions;
//   softmax        a lane holds 8 scores of one row;
//   O^T += V^T P   the lane's probabilities are the B operand as they are.
// Both products read their operands from memory to registers as they lie: a key's
// dimensions are consecutive, and so are 8 positions of a value's dimension.  Block t's
// row 4 c + i is position 8 c + 4 t + i, so that a lane's scores of both blocks are the 8
// consecutive positions that its lane of the value operand holds.
//
// One token per sequence is bound by the cache's bytes, 8 KV heads of 128 and 4 query heads
// each: 64 sequences of 150 to 8000 196 to 203 us (1.07 GB, 5.3 to 5.5 TB/s; a large read
// reaches 6.2), 64 of 2000 91 us (5.8), and, of few positions, by memory's latency: one text
// of 701 9.8 us in two launches.  A wave's products are 8 times as fast as its bytes come, so
// the 4 rows of 16 that it uses cost nothing.
constexpr int kTile = 32;
constexpr int NW = 4;  // waves of a workgroup
// Workgroups per CU that the positions are shared out to, and that the registers hold at
// least.  (Three of 128 dimensions spill: one text of 31777 43 us, two 33.)
constexpr int resident(long hd) { return hd == 256 ? 1 : 2; }
// The same of runs by blocks.  (Of 64 dimensions, two / three: 8 of 1000 rows after 3000 261 /
// 245 us.)
constexpr int resident_blocks(long hd) { return hd == 64 ? 3 : resident(hd); }
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are 2^8 times the softmax's, relative to a maximum that follows the true
// one only when it lags by 2^6: below 2^14, so fp16 holds them, and those down to 2^-22
// of the largest are normal numbers.  The matrix instruction multiplies numbers of the
// cache's type with the values, so a probability goes in as two: itself rounded, and what
// that left (in all 2^-22 of it is lost in fp16, 2^-16 in bf16).  The second product costs
// nothing where the bytes are the bound, and runs by blocks a third (chunks of prompts 147 us
// without it, 191 with it); without it they would be off by more than the result's own
// rounding (relative to 64 bits 2.7e-4, 2.1e-4 with it, in fp16; 2.1e-3 and 1.7e-3 in bf16).
// A row's sum is of the probabilities as they are, in fp32.
constexpr float kUp = 8.f, kLag = 6.f;
// Positions that workgroups share out as one.
constexpr int kGrain = 128;
// Positions that a share of a block's has at least.  (80 rows of one sequence of 1020: 19.6
// us, in one share 43.)
constexpr long kShare = 256;

template <class T>
struct Attend {
  Step P;
  const T *q, *k, *v;
  T* out;
  // entries of the workspace: R (of blocks: 128) rows of HD sums each, then of as many
  // (maximum, sum)
  float* part;
  long ld_q, ld_o;
  int rep, max_new, R, wgs;
  int shares, each;  // of a block's positions, and the stages of one
  long entries;
  float scale;
};

// f over the four lanes, 16 apart, that hold one row
template <class F>
__device__ __forceinline__ float over_row(float x, F f) {
  const uint32_t w = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  x = f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  const uint32_t v = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float row_max(float x) {
  return over_row(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float row_sum(float x) {
  return over_row(x, [](float a, float b) { return a + b; });
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// A sequence's rows [row, row + n) of the step, its cached positions C and the end L of
// those that are read.  Positions past the table's are all one to a row that sees them,
// so neither C nor L exceeds the first of them by more than 1.  none: rows that are zero
// (no part); nan: NaN (more than max_new).
struct Run {
  int row, n, C, L;
  bool none, nan;
};
template <class T>
__device__ __forceinline__ Run run_of(const Attend<T>& A, int b) {
  const Step& P = A.P;
  Run r = {b, 1, 0, 0, false, false};
  if (P.starts) {
    r.row = min(max(P.starts[b], 0), P.T);
    r.n = max(min(P.starts[b + 1], P.T) - r.row, 0);
  }
  const long C = P.lens[b];
  const int cap = (int)(P.cols * P.page);
  r.none = C < 0, r.nan = !r.none && r.n > A.max_new;
  if (r.n == 0 || r.none || r.nan) return r;
  r.C = C > cap ? cap + 1 : (int)C;
  r.L = min(r.C + r.n, cap + 1);
  return r;
}

// The rows of a run that none attends for, of KV head g; and of no run.
template <class T, int HD>
__device__ __forceinline__ void fill(const Attend<T>& A, const Run& r, int g, int part, int parts) {
  const T x = (T)(r.nan ? __builtin_nanf("") : 0.f);
  typename Vec<T>::t y;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = x;
  const int cols = A.rep * (HD / 8);
  for (long i = (long)part * blockDim.x + threadIdx.x; i < (long)r.n * cols;
       i += (long)parts * blockDim.x) {
    const int t = (int)(i / cols), c = (int)(i - (long)t * cols);
    *reinterpret_cast<typename Vec<T>::t*>(A.out + (long)(r.row + t) * A.ld_o +
                                           (long)g * A.rep * HD + 8 * c) = y;
  }
}

template <class T, int HD>
__device__ __forceinline__ void fill_rest(const Attend<T>& A, int g, int part, int parts) {
  if (!A.P.starts) return;
  const int first = min(max(A.P.starts[0], 0), A.P.T), end = min(max(A.P.starts[A.P.B], first), A.P.T);
  fill<T, HD>(A, Run{0, first, 0, 0, true, false}, g, part, parts);
  fill<T, HD>(A, Run{end, A.P.T - end, 0, 0, true, false}, g, part, parts);
}

// Sums of the lanes up to each (row_shr:1, 2, 4, 8, then row_bcast:15, 31).
__device__ __forceinline__ int lane_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);
  return x;
}

template <class T>
__device__ __forceinline__ int grains_of(const Attend<T>& A, int b) {
  return (run_of(A, b).L + kGrain - 1) / kGrain;
}

// The grains of all (sequence, KV head) pairs in order, dealt evenly: the first `more` of
// wgs workgroups take each + 1 of them.
struct Deal {
  int wgs, each, more;
  __device__ Deal(int total, int most) : wgs(min(total, most)) {
    each = wgs ? total / wgs : 0, more = total - each * wgs;
  }
  __device__ int from(int w) const { return w * each + min(w, more); }
  __device__ int owner(int x) const {
    const int big = more * (each + 1);
    return x < big ? x / (each + 1) : more + (x - big) / each;
  }
};

// Grains of one head of the sequences below `to`, by a wave.
template <class T>
__device__ __forceinline__ int grains_below(const Attend<T>& A, int to) {
  int n = 0;
  for (int b = threadIdx.x & 63; b < to; b += 64) n += grains_of(A, b);
  return __builtin_amdgcn_readlane(lane_scan(n), 63);
}

// Values that are no numbers.  A row has the infinities and NaN of the positions that it
// sees in their dimensions, whatever their weights: a softmax's are above 0.  A product
// makes NaN of an infinity where the probability was rounded to 0, or with what its rounding
// left (of either sign, or 0), also for the rows that do not see it.  So at positions that
// only some rows see (past lo) they are taken out of the products and added to the rows
// afterwards.  Among the positions that all rows see a first walk looks for none: its sums
// tell whether there was one (far), and then a second walk takes them out everywhere (lo =
// -1).  The joins' weights are not 0 either (weight).  The look at the sums costs 0.2 to 0.3
// us of a launch, 2 to 3 % of prompts by blocks.
//
// Values near bf16's largest: 2^14 times one is no number of fp32.  Their sums are found in the
// same way, and the second walk's probabilities are 2^40 times smaller (Vec::less; a factor
// behind the exponential, so that other rows' sums come out as they were; in bf16 3 % of
// prompts by blocks).
//
// Of 8 positions from `at` on, the values that must not reach a product: those at positions
// past hi, which no row sees (their probabilities are zero, but what lies there may be
// anything), and those past lo that are no numbers.  Returns whether there was one of the
// latter.
template <class T, int E>
__device__ __forceinline__ uint32_t clean(typename Vec<T>::t (&v)[E], int at, int lo, int hi) {
  uint32_t odd = 0;
  asm volatile("" : "+v"(at));  // (nothing of this stays in registers where it is not used)
#pragma unroll
  for (int e = 0; e < E; ++e) {
    u32x4 w = __builtin_bit_cast(u32x4, v[e]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int p = at + 2 * c;
      w[c] &= (p <= hi ? 0xffffu : 0u) | (p + 1 <= hi ? 0xffff0000u : 0u);
      const uint32_t m = (p > lo && (w[c] & Vec<T>::inf) == Vec<T>::inf ? 0xffffu : 0u) |
                         (p + 1 > lo && (w[c] >> 16 & Vec<T>::inf) == Vec<T>::inf ? 0xffff0000u : 0u);
      odd |= m, w[c] &= ~m;
    }
    v[e] = __builtin_bit_cast(typename Vec<T>::t, w);
  }
  return odd;
}

// Those of positions [from, to], added to the rows that see them.
template <class T, int HD, int NT>
__device__ __forceinline__ void add_odd(const Attend<T>& A, float4v (&o)[NT][HD / 16],
                                        const int (&lim)[NT], int b, int g, int from, int to,
                                        int kg) {
  const Step& P = A.P;
  for (int p = from; p <= to; ++p) {
    const long id = page_of(P, b, p);
    if (id < 0) continue;
    const int slot = p & (P.page - 1);
    const T* v = A.v + ((id * P.nkv + g) * P.page + (slot & ~7)) * HD + (slot & 7);
#pragma unroll
    for (int e = 0; e < HD / 16; ++e)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float x = (float)v[8 * (16 * e + 4 * kg + c)];
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if (p <= lim[t] && !(__builtin_fabsf(x) < __builtin_inff())) o[t][e][c] += x;
      }
  }
}

// Whether one of a row's sums is no number, or past about kFar, so that a join might overflow.
constexpr float kFar = 0x1p100f;
template <int N>
__device__ __forceinline__ bool far(const float4v (&o)[N]) {
  float4v x = (float4v)(0.f);
#pragma unroll
  for (int e = 0; e < N; ++e)
#pragma unroll
    for (int c = 0; c < 4; ++c) x[c] = __builtin_fmaf(o[e][c], 0x1p127f / kFar, x[c]);
  return !(__builtin_fabsf((x[0] + x[1]) + (x[2] + x[3])) < __builtin_inff());
}

// The weight 2^x of sums in a join: above 0, so that an infinity stays one.  (2^-149 times any
// finite sum is below 2^-21.)
__device__ __forceinline__ float weight(float x) {
  return fmaxf(__builtin_amdgcn_exp2f(x), 0x1p-149f);
}

// The sums of NT x 16 rows over a wave's positions.
template <class T, int HD, int NT>
struct Sums {
  float4v o[NT][HD / 16];
  float mx[NT], l[NT];  // (l while a walk runs: of the lane's positions)
  __device__ __forceinline__ void start(int t) {
    mx[t] = -__builtin_inff();
    l[t] = 0.f;
#pragma unroll
    for (int e = 0; e < HD / 16; ++e) o[t][e] = (float4v)(0.f);
  }
  // The sums so far are `less` times what they are: a row's are brought back, or, where one
  // is past kFar, they are what they are to a larger maximum.
  __device__ __forceinline__ void end(float less) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      l[t] = row_sum(l[t]);
      if (less == 1.f) continue;
      const float up = 1.f / less, most = kFar * less;
      float over = 0.f;
#pragma unroll
      for (int e = 0; e < HD / 16; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float x = __builtin_fabsf(o[t][e][c]);
          if (x >= most && x < __builtin_inff()) over = 1.f;
        }
      if (row_max(over) > 0.f) {
        mx[t] += __builtin_log2f(up);
      } else {
        l[t] *= up;
#pragma unroll
        for (int e = 0; e < HD / 16; ++e) o[t][e] *= up;
      }
    }
  }
};

// A wave's tiles `wave`, `wave` + NW, .. of [first, end) of a run, for rows row0 on of KV
// head g.  All rows see the positions up to lo, none sees past hi.  The next tile's keys
// are asked for when this one's scores are there, its values after this one's product:
// about a tile is in flight throughout, in the registers of one.
template <class T, int HD, int NT>
__device__ __forceinline__ void walk(const Attend<T>& A, Sums<T, HD, NT>& W, const Run& r, int b,
                                     int g, int row0, int first, int end, int lo, int hi, int wave,
                                     int lane) {
  typedef typename Vec<T>::t V8;
  const Step& P = A.P;
  const int shift = __builtin_ctz(P.page), mask = P.page - 1, n = lane & 15, kg = lane >> 4;
  V8 q[NT][HD / 32];
  int lim[NT];  // the last position that this lane's row sees
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = row0 + 16 * t + n, tok = row / A.rep, head = row - tok * A.rep;
    const bool in = row < A.rep * r.n;
    const T* src = A.q + (long)(r.row + tok) * A.ld_q + (long)(g * A.rep + head) * HD + 8 * kg;
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
      u32x4 w = {0, 0, 0, 0};
      if (in) w = *reinterpret_cast<const u32x4*>(src + 32 * u);
      q[t][u] = __builtin_bit_cast(V8, w);
    }
    lim[t] = in ? r.C + tok : lo;
    W.start(t);
  }
  const int tiles = (min(end, hi + 1) - first + kTile - 1) / kTile;
  const int mine = (tiles - wave + NW - 1) / NW;
  if (mine <= 0) return;
  auto start = [&](int i) { return first + kTile * (wave + NW * min(i, mine - 1)); };
  // The pages of a tile's halves of 16 positions as this lane has them: of its key rows
  // and of its values.
  const int* table = P.table + (long)b * P.ld;
  struct Ids {
    int k, v;
  };
  auto ids = [&](int i) {
    const int p0 = start(i);
    const int ck = (p0 + 8 * (n >> 2)) >> shift, cv = (p0 + 8 * kg) >> shift;
    return Ids{ck < P.cols ? table[ck] : -1, cv < P.cols ? table[cv] : -1};
  };
  auto named = [&](int id) { return id >= 0 && id < P.pages; };
  auto base = [&](const T* x, int id) {
    return x + ((long)(named(id) ? id : 0) * P.nkv + g) * P.page * HD;
  };
  V8 k[2][HD / 32], v[HD / 16];
  auto keys = [&](int i, int id) {
    const T* x = base(A.k, id) + ((start(i) + 8 * (n >> 2) + (n & 3)) & mask) * HD + 8 * kg;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int u = 0; u < HD / 32; ++u)
        k[j][u] = *reinterpret_cast<const V8*>(x + 4 * j * HD + 32 * u);
  };
  auto values = [&](int i, int id) {
    const T* x = base(A.v, id) + ((start(i) + 8 * kg) & mask) * HD + 8 * n;
#pragma unroll
    for (int e = 0; e < HD / 16; ++e) v[e] = *reinterpret_cast<const V8*>(x + 128 * e);
  };
  const float scale = A.scale * kLog2e;

  // apart: values that are no numbers are taken out at every position
  for (bool apart = false;; apart = true) {
    asm volatile("" : "+s"(first), "+s"(g));  // (else what both walks begin with stays in registers)
    const int all = apart ? -1 : lo;
    const float less = apart ? Vec<T>::less : 1.f;
    int odd_from = mine, odd_to = -1;  // the tiles that had some of those
    Ids id = ids(0), next = ids(1);
    keys(0, id.k);
    values(0, id.v);
    for (int i = 0; i < mine; ++i) {
      const Ids after = ids(i + 2);
      const int p0 = start(i), at = p0 + 8 * kg;  // this lane's 8 positions
      const bool bad = !named(id.v);              // they lie on no page
      const bool edge = p0 + kTile - 1 > all || __any(bad);
      float4v s[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[t][j] = (float4v)(0.f);
#pragma unroll
          for (int u = 0; u < HD / 32; ++u) s[t][j] = Vec<T>::mfma(k[j][u], q[t][u], s[t][j]);
        }
      keys(i + 1, next.k);
      V8 p[NT], rest[NT];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (edge)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (bad) s[t][j][c] = __builtin_nanf("");
              if (at + 4 * j + c > lim[t]) s[t][j][c] = -__builtin_inff();
            }
        float tm = s[t][0][0];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) tm = fmaxf(tm, s[t][j][c]);
        if (__any(tm * scale > W.mx[t] + kLag)) {
          const float nm = fmaxf(W.mx[t], row_max(tm) * scale);
          const float al = nm == W.mx[t] ? 1.f : __builtin_amdgcn_exp2f(W.mx[t] - nm);
          W.l[t] *= al;
#pragma unroll
          for (int e = 0; e < HD / 16; ++e) W.o[t][e] *= al;
          W.mx[t] = nm;
        }
        const float ref = W.mx[t] == -__builtin_inff() ? 0.f : W.mx[t] - kUp;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j][c], scale, -ref));
            if (Vec<T>::less != 1.f) x *= less;
            W.l[t] += x;
            p[t][4 * j + c] = (T)x;
            rest[t][4 * j + c] = (T)(x - (float)p[t][4 * j + c]);
          }
      }
      // (values on no page were read from another one: no row gets a number that it sees)
      if (edge && __any(clean<T>(v, bad ? hi + 1 : at, all, hi)))
        odd_from = min(odd_from, i), odd_to = i;
#pragma unroll
      for (int e = 0; e < HD / 16; ++e)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          W.o[t][e] = Vec<T>::mfma(v[e], p[t], W.o[t][e]);
          W.o[t][e] = Vec<T>::mfma(v[e], rest[t], W.o[t][e]);
        }
      values(i + 1, next.v);
      id = next, next = after;
    }
    bool odd = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      odd |= row0 + 16 * t + n < A.rep * r.n && far(W.o[t]);
    }
    if (!apart && __any(odd)) {
#pragma unroll
      for (int t = 0; t < NT; ++t) W.start(t);
      continue;
    }
    for (int i = odd_from; i <= odd_to; ++i)
      add_odd<T, HD, NT>(A, W.o, lim, b, g, max(start(i), all + 1), min(start(i) + kTile - 1, hi),
                         kg);
    W.end(less);
    break;
  }
}

// The waves' sums of 16 rows joined, then the rows themselves, or the range's entry of
// the workspace.
template <class T, int HD, int NT>
__device__ __forceinline__ void finish(const Attend<T>& A, const Sums<T, HD, NT>& W, const Run& r,
                                       int g, int row0, long entry, float* s_o, float* s_m,
                                       int wave, int lane) {
  constexpr int kPad = HD + 4;
  const int n = lane & 15, kg = lane >> 4, rows = A.rep * r.n;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    __syncthreads();  // (the last use of the buffers)
    if (row0 + 16 * t + n < rows) {
      if (kg == 0) s_m[(wave * 16 + n) * 2] = W.mx[t], s_m[(wave * 16 + n) * 2 + 1] = W.l[t];
#pragma unroll
      for (int e = 0; e < HD / 16; ++e)
        *reinterpret_cast<float4v*>(s_o + (wave * 16 + n) * kPad + 16 * e + 4 * kg) = W.o[t][e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (HD / 8); i += 64 * NW) {
      const int rr = i / (HD / 8), d = 8 * (i % (HD / 8)), row = row0 + 16 * t + rr;
      if (row >= rows) continue;
      float m = -__builtin_inff();
#pragma unroll
      for (int w = 0; w < NW; ++w) m = fmaxf(m, s_m[(w * 16 + rr) * 2]);
      const float ref = m == -__builtin_inff() ? 0.f : m;
      float sum = 0.f, x[8] = {};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        // (a wave without tiles has sums of zero)
        const float al = weight(s_m[(w * 16 + rr) * 2] - ref);
        sum += al * s_m[(w * 16 + rr) * 2 + 1];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += al * s_o[(w * 16 + rr) * kPad + d + j];
      }
      if (entry < 0) {
        const int tok = row / A.rep, head = row - tok * A.rep;
        const float is = 1.f / sum;
        typename Vec<T>::t y;
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = (T)(x[j] * is);
        *reinterpret_cast<typename Vec<T>::t*>(A.out + (long)(r.row + tok) * A.ld_o +
                                               (long)(g * A.rep + head) * HD + d) = y;
      } else {
        const long at = entry * A.R + row;
#pragma unroll
        for (int j = 0; j < 8; j += 4)
          *reinterpret_cast<float4v*>(A.part + at * HD + d + j) =
              float4v{x[j], x[j + 1], x[j + 2], x[j + 3]};
        float* pm = A.part + 2 * (long)A.wgs * A.R * HD + at * 2;
        if (d == 0) pm[0] = m, pm[1] = sum;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Runs of many rows.  A workgroup of 4 waves takes 128 rows of one (sequence, KV head), 32
// a wave, and walks the positions in stages that all four read from LDS; the next stage
// goes from memory to LDS (buffer_load ... lds) meanwhile.  A stage lies there as in the
// pages, but that a key's 16-byte chunks are at chunk ^ key(position), so that the 16
// positions that a read takes cover the banks once (the counter of conflicts stays at 0).
// Two workgroups per CU: one's loads and softmax under the other's products.
//
// Bounds: where there are several workgroups for each place, the matrix units, which make a
// half more products than the formula has, the second one for what a probability's rounding
// left (4000 rows after 4000 positions: 530 to 550 us, 0.72 to 0.74 PFLOP/s of the formula's
// and 1.1 in all, a large product reaches 1.14 to 1.17); where each has about one, the longest
// block's stages after each other while others are done: runs of 1000, 688 and 376 after 900
// to 4000 187 to 192 us.
// Measured without the second product (391 and 146 us then) and not taken: all blocks' stages
// dealt evenly to the workgroups (they then walk different positions at once, out of L2: 462
// us, with a plan and joins of 23); five smaller stages in LDS, four of them on their way, and
// scores made a stage ahead beside the exponentials (no difference); more shares than places
// (146 to 201).
constexpr int kBlock = 128;
constexpr int stage_of(int hd) { return hd == 256 ? 32 : 64; }

// The blocks of a run, and the stages of one: up to the last position that its rows see.
template <class T>
__device__ __forceinline__ int blocks_of(const Attend<T>& A, const Run& r) {
  return r.L ? (A.rep * r.n + kBlock - 1) / kBlock : 0;
}
template <class T, int HD>
__device__ __forceinline__ int stages_of(const Attend<T>& A, const Run& r, int block) {
  const int top = r.C + min((block * kBlock + kBlock - 1) / A.rep, r.n - 1);
  return min(top, r.L - 1) / stage_of(HD) + 1;
}

// Stages [from, to) of a block: its rows, or, with entry >= 0, their sums to the workspace.
template <class T, int HD>
__device__ __forceinline__ void block_range(const Attend<T>& A, const Run& r, int b, int g,
                                            int block, int from, int to, long entry,
                                            unsigned char* s_buf) {
  typedef typename Vec<T>::t V8;
  constexpr int SP = stage_of(HD), NT = 2, kChunks = HD / 8;  // 16-byte chunks of a key
  constexpr int kBytes = SP * HD * 2;      // of a stage's keys, and of its values
  constexpr int kPos = 64 / kChunks;       // keys per DMA instruction
  constexpr int kDma = kBytes / 1024 / 4;  // instructions per wave and operand
  const Step& P = A.P;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int n = lane & 15, kg = lane >> 4;
  const int rows = A.rep * r.n, row0 = block * kBlock + 32 * wave;
  const bool busy = row0 < rows;

  V8 q[NT][HD / 32];
  int lim[NT];
  // positions that all of this wave's rows see, and past which none sees any
  const int lo = r.C + row0 / A.rep;
  const int hi = min(r.C + min((row0 + 31) / A.rep, r.n - 1), r.L - 1);
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = row0 + 16 * t + n, tok = row / A.rep, head = row - tok * A.rep;
    const bool in = row < rows;
    const T* src = A.q + (long)(r.row + tok) * A.ld_q + (long)(g * A.rep + head) * HD + 8 * kg;
#pragma unroll
    for (int u = 0; u < HD / 32; ++u) {
      u32x4 w = {0, 0, 0, 0};
      if (in) w = *reinterpret_cast<const u32x4*>(src + 32 * u);
      q[t][u] = __builtin_bit_cast(V8, w);
    }
    lim[t] = in ? r.C + tok : lo;
  }

  const int shift = __builtin_ctz(P.page);
  // The pages of a stage's positions by sixteens (-1: none): scalars, read ahead through
  // the scalar cache, so that no wait for them is one for the stage on its way.
  typedef const __attribute__((address_space(4))) int* Table;
  const Table table = (Table)(uintptr_t)(P.table + (long)b * P.ld);
  struct Ids {
    int id[SP / 16];
  };
  const bool one = P.page >= SP;  // a stage lies on one page
  auto pages = [&](int st) {
    Ids x;
    auto at = [&](int i) {
      const int col = (st * SP + 16 * i) >> shift;
      const int id = col < P.cols ? table[col] : -1;
      return id >= 0 && id < P.pages ? id : -1;
    };
    x.id[0] = at(0);
#pragma unroll
    for (int i = 1; i < SP / 16; ++i) x.id[i] = one ? x.id[0] : at(i);
    return x;
  };
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)s_buf;
  // DMA: instruction i of wave w moves KB w + 4 i of a stage's keys and of its values.  A
  // page that is not there reads as zero (a descriptor of no bytes).
  const int head_bytes = P.page * HD * 2;
  const long page_elems = (long)P.nkv * P.page * HD, head = (long)g * P.page * HD;
  const T *keys0 = A.k + head, *values0 = A.v + head;
  auto issue = [&](int st, const Ids& x) {
    const uint32_t at = lds0 + (uint32_t)(st & 1) * 2 * kBytes + wave * 1024;
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      // the page of instruction i's positions, kPos * (wave + 4 i) on (or the 8 around them)
      const int j = kPos * 4 * i / 16;
      const int id = kPos == 8 && wave >> 1 ? x.id[j + (kPos == 8)] : x.id[j];
      const long page = max(id, 0) * page_elems;
      const int bytes = id < 0 ? 0 : head_bytes;
      const int kp = kPos * (wave + 4 * i), pos = kp + lane / kChunks;  // within the stage
      const int m = ((pos >> 3) & 3) * 4 + (pos & 3), key = kChunks == 8 ? m >> 1 : m;
      dma_b128(rsrc(keys0 + page, bytes),
               (lane / kChunks) * HD * 2 + 16 * ((lane % kChunks) ^ key),
               (uint32_t)((st * SP + kp) & (P.page - 1)) * HD * 2, at + i * 4096);
      // KB kb of the values: 512 / HD positions' worth, in slots of 8
      const int kb = wave + 4 * i, vp = kb * 512 / HD & ~7;
      dma_b128(rsrc(values0 + page, bytes), 16 * lane,
               (uint32_t)((st * SP + vp) & (P.page - 1)) * HD * 2 + (kb * 1024) % (16 * HD),
               at + kBytes + i * 4096);
    }
  };

  // this lane's part of the reads
  uint32_t k_at[HD / 32];
  const int mine = kChunks == 8 ? n >> 1 : n;
#pragma unroll
  for (int u = 0; u < HD / 32; ++u)
    k_at[u] = lds0 + (8 * (n >> 2) + (n & 3)) * HD * 2 + 16 * ((4 * u + kg) ^ mine);
  const uint32_t v_at = lds0 + kBytes + kg * HD * 16 + n * 16;
  const float scale = A.scale * kLog2e;

  __shared__ int s_again;  // (set and read between the stages' barriers and the one behind them)
  if (tid == 0) s_again = 0;
  Sums<T, HD, NT> W;
  for (bool apart = false;; apart = true) {
    asm volatile("" : "+s"(from));  // (as in walk)
    const int all = apart ? -1 : lo;
    const float less = apart ? Vec<T>::less : 1.f;
    int odd_from = to, odd_to = -1;  // the stages that had values which are no numbers
#pragma unroll
    for (int t = 0; t < NT; ++t) W.start(t);
    Ids id = pages(from), next = pages(from + 1);
    issue(from, id);
    for (int st = from; st < to; ++st) {
      wait_vmcnt<0>();  // this wave's part of the stage has landed
      stage_barrier();  // everyone's, and the stage before is used
      if (st + 1 < to) issue(st + 1, next);
      uint32_t bad = 0;
#pragma unroll
      for (int i = 0; i < SP / 16; ++i) bad |= id.id[i] < 0 ? 1u << i : 0u;
      id = next, next = pages(st + 2);
      const uint32_t here = (uint32_t)(st & 1) * 2 * kBytes;
      // (Waves without rows, or past the last position that theirs see, go along.)
      const bool edge = st * SP + SP - 1 > all || bad;
      const int p0 = st * SP;
      float4v s[NT][SP / 16];  // block 2 h + j of half h
#pragma unroll
      for (int x = 0; x < SP / 16; ++x) {
        V8 k[HD / 32];
#pragma unroll
        for (int u = 0; u < HD / 32; ++u)
          k[u] = lds_read<V8>(k_at[u] + here + (32 * (x >> 1) + 4 * (x & 1)) * HD * 2);
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][x] = (float4v)(0.f);
#pragma unroll
        for (int u = 0; u < HD / 32; ++u)
#pragma unroll
          for (int t = 0; t < NT; ++t) s[t][x] = Vec<T>::mfma(k[u], q[t][u], s[t][x]);
      }
      V8 p[NT][SP / 32], rest[NT][SP / 32];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if (edge) {
          int see = lim[t] - p0 - 8 * kg;
          asm volatile("" : "+v"(see));  // (else as many differences from it stay in registers)
#pragma unroll
          for (int x = 0; x < SP / 16; ++x) {
            const bool none = bad >> (2 * (x >> 1) + (kg >> 1)) & 1;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if (none) s[t][x][c] = __builtin_nanf("");
              if (32 * (x >> 1) + 4 * (x & 1) + c > see) s[t][x][c] = -__builtin_inff();
            }
          }
        }
        float tm = s[t][0][0];
#pragma unroll
        for (int x = 0; x < SP / 16; ++x)
#pragma unroll
          for (int c = 0; c < 4; ++c) tm = fmaxf(tm, s[t][x][c]);
        if (__any(tm * scale > W.mx[t] + kLag)) {
          const float nm = fmaxf(W.mx[t], row_max(tm) * scale);
          const float al = nm == W.mx[t] ? 1.f : __builtin_amdgcn_exp2f(W.mx[t] - nm);
          W.l[t] *= al;
#pragma unroll
          for (int e = 0; e < HD / 16; ++e) W.o[t][e] *= al;
          W.mx[t] = nm;
        }
        const float ref = W.mx[t] == -__builtin_inff() ? 0.f : W.mx[t] - kUp;
#pragma unroll
        for (int x = 0; x < SP / 16; ++x)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][x][c], scale, -ref));
            if (Vec<T>::less != 1.f) y *= less;
            const int i = 4 * (x & 1) + c;
            W.l[t] += y;
            p[t][x >> 1][i] = (T)y;
            rest[t][x >> 1][i] = (T)(y - (float)p[t][x >> 1][i]);
          }
      }
#pragma unroll
      for (int h = 0; h < SP / 32; ++h) {
#pragma unroll
        for (int e0 = 0; e0 < HD / 16; e0 += 4) {
          V8 v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = lds_read<V8>(v_at + here + h * HD * 64 + (e0 + e) * 256);
          if (edge && __any(clean<T>(v, p0 + 32 * h + 8 * kg, all, hi)))
            odd_from = min(odd_from, st), odd_to = st;
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              W.o[t][e0 + e] = Vec<T>::mfma(v[e], p[t][h], W.o[t][e0 + e]);
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < NT; ++t)
              W.o[t][e0 + e] = Vec<T>::mfma(v[e], rest[t][h], W.o[t][e0 + e]);
        }
      }
    }
    if (!apart) {
      bool odd = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        odd |= row0 + 16 * t + n < rows && far(W.o[t]);
      }
      if (__any(odd)) s_again = 1;
      __syncthreads();  // (also: the last stage is used, before the first of a second walk)
      if (s_again) continue;
    }
    if (busy)
      add_odd<T, HD, NT>(A, W.o, lim, b, g, max(odd_from * SP, all + 1),
                         min(odd_to * SP + SP - 1, hi), kg);
    W.end(less);
    break;
  }
  if (!busy) return;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int row = row0 + 16 * t + n, tok = row / A.rep, head = row - tok * A.rep;
    if (row >= rows) continue;
    if (entry >= 0) {
      const long at = entry * kBlock + (row - block * kBlock);
      float* dst = A.part + at * HD + 4 * kg;
#pragma unroll
      for (int e = 0; e < HD / 16; ++e) *reinterpret_cast<float4v*>(dst + 16 * e) = W.o[t][e];
      float* pm = A.part + A.entries * kBlock * HD + at * 2;
      if (kg == 0) pm[0] = W.mx[t], pm[1] = W.l[t];
      continue;
    }
    const float is = 1.f / W.l[t];
    T* dst = A.out + (long)(r.row + tok) * A.ld_o + (long)(g * A.rep + head) * HD + 4 * kg;
#pragma unroll
    for (int e = 0; e < HD / 16; ++e) {
      typedef T V4 __attribute__((ext_vector_type(4)));
      V4 y;
#pragma unroll
      for (int c = 0; c < 4; ++c) y[c] = (T)(W.o[t][e][c] * is);
      *reinterpret_cast<V4*>(dst + 16 * e) = y;
    }
  }
}

// A workgroup per (KV head, block and share of its positions, sequence), the longest blocks
// of a run first.  A head's blocks side by side walk the same positions at once, so all but
// the first find them in the XCD's L2: with the sequences side by side instead, 8 of 1000
// rows after 3000 take 635 us, as it is 390.  A block's A.each stages a share (the rest in
// the last); its entry of the workspace goes by the block and the share.
template <class T, int HD>
__global__ __launch_bounds__(256, resident_blocks(HD)) void block_kernel(Attend<T> A) {
  __shared__ __align__(1024) unsigned char s_buf[8 * stage_of(HD) * HD];
  const int g = blockIdx.x, b = blockIdx.z, part = gridDim.y - 1 - blockIdx.y;
  const int block = part / A.shares, share = part - block * A.shares;
  const Run r = run_of(A, b);
  if (b == 0) fill_rest<T, HD>(A, g, part, gridDim.y);
  if (r.none || r.nan) return fill<T, HD>(A, r, g, part, gridDim.y);
  if (block >= blocks_of(A, r)) return;
  const int stages = stages_of<T, HD>(A, r, block), from = share * A.each;
  if (from >= stages) return;
  const int to = share == A.shares - 1 ? stages : min(from + A.each, stages);
  const long entry = (((long)b * A.P.nkv + g) * gridDim.y) + part;
  block_range<T, HD>(A, r, b, g, block, from, to, to - from == stages ? -1 : entry, s_buf);
}

// The entries of a block's shares joined, 1024 / HD rows at a time.  Grid (nkv, blocks *
// HD / 8, B).
template <class T, int HD>
__global__ __launch_bounds__(256) void join_blocks_kernel(Attend<T> A) {
  constexpr int kAcross = HD / 4, kRows = 256 / kAcross;
  const int g = blockIdx.x, b = blockIdx.z, block = blockIdx.y / (HD / 8);
  const Run r = run_of(A, b);
  if (block >= blocks_of(A, r)) return;
  const int stages = stages_of<T, HD>(A, r, block);
  const int n = min((stages + A.each - 1) / A.each, A.shares);
  const int c = threadIdx.x % kAcross;
  const int in = blockIdx.y % (HD / 8) * kRows + threadIdx.x / kAcross, row = block * kBlock + in;
  if (n < 2 || row >= A.rep * r.n) return;
  const long blocks = gridDim.y / (HD / 8), first = (((long)b * A.P.nkv + g) * blocks + block) * A.shares;
  const float* ms = A.part + A.entries * kBlock * HD;
  float m = -__builtin_inff(), sum = 0.f;
  float4v o = (float4v)(0.f);
  for (int i = 0; i < n; i += 4) {
    float em[4], el[4];
    float4v eo[4];  // four entries asked for together
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const long e = (first + min(i + j, n - 1)) * kBlock + in;
      em[j] = ms[2 * e], el[j] = ms[2 * e + 1];
      eo[j] = *reinterpret_cast<const float4v*>(A.part + e * HD + 4 * c);
    }
    float nm = m;
#pragma unroll
    for (int j = 0; j < 4; ++j) nm = fmaxf(nm, em[j]);
    const float ref = nm == -__builtin_inff() ? 0.f : nm;
    const float a = weight(m - ref);
    o *= a, sum *= a, m = nm;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i + j >= n) continue;
      const float z = weight(em[j] - ref);
      o += eo[j] * z, sum += el[j] * z;
    }
  }
  const int tok = row / A.rep, head = row - tok * A.rep;
  const float is = 1.f / sum;
  typedef T V4 __attribute__((ext_vector_type(4)));
  V4 y;
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = (T)(o[j] * is);
  *reinterpret_cast<V4*>(A.out + (long)(r.row + tok) * A.ld_o + (long)(g * A.rep + head) * HD +
                         4 * c) = y;
}

// A workgroup per (KV head, block of 16 NT rows, sequence), over all of its positions.
template <class T, int HD, int NT>
__global__ __launch_bounds__(64 * NW, resident(HD)) void whole_kernel(Attend<T> A) {
  __shared__ __align__(16) float s_o[NW * 16 * (HD + 4)];
  __shared__ float s_m[NW * 16 * 2];
  const int g = blockIdx.x, b = blockIdx.z, row0 = (gridDim.y - 1 - blockIdx.y) * 16 * NT;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const Run r = run_of(A, b);
  if (b == 0) fill_rest<T, HD>(A, g, blockIdx.y, gridDim.y);
  if (r.none || r.nan) return fill<T, HD>(A, r, g, blockIdx.y, gridDim.y);
  if (row0 >= A.rep * r.n) return;
  Sums<T, HD, NT> W;
  const int last = min((row0 + 16 * NT - 1) / A.rep, r.n - 1);
  const int lo = r.C + row0 / A.rep, hi = min(r.C + last, r.L - 1);
  walk<T, HD, NT>(A, W, r, b, g, row0, 0, r.L, lo, hi, wave, lane);
  finish<T, HD, NT>(A, W, r, g, row0, -1, s_o, s_m, wave, lane);
}

// The grains of all (sequence, KV head) pairs in order, an even share of them for each
// workgroup, wherever the sequences' borders are: one range of positions of one head, or
// several.  A head's range that is not whole leaves its sums in the workspace, in entry
// 2 w of workgroup w, or 2 w + 1 if it is not w's first, for join_kernel.
template <class T, int HD, int NT>
__global__ __launch_bounds__(64 * NW, resident(HD)) void share_kernel(Attend<T> A) {
  __shared__ __align__(16) float s_o[NW * 16 * (HD + 4)];
  __shared__ float s_m[NW * 16 * 2];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), w = blockIdx.x;
  const int nkv = A.P.nkv;
  const Deal D(uniform(grains_below(A, A.P.B)) * nkv, A.wgs);
  const int from = D.from(w);
  int left = w < D.wgs ? D.from(w + 1) - from : 0, b = 0, g = 0, at = 0, n = 0;
  int base = 0;  // grains of one head of the sequences before
  for (int c = 0; c < A.P.B && left; c += 64) {
    const int t = c + lane < A.P.B ? grains_of(A, c + lane) : 0;
    const int sum = lane_scan(t);
    const unsigned long long past = __ballot((base + sum) * nkv > from);
    if (past) {
      const int i = __builtin_ctzll(past);
      b = c + i;
      n = __builtin_amdgcn_readlane(t, i);
      const int in = from - (base + __builtin_amdgcn_readlane(sum, i) - n) * nkv;
      g = in / n, at = in - g * n;
      break;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  for (bool start = true; left > 0; start = false) {
    while (at >= n) {  // the next head that has grains
      at = 0;
      if (n > 0 && ++g < nkv) break;
      g = 0;
      if (++b >= A.P.B) return;  // (cannot be: the grains left are of some head)
      n = uniform(grains_of(A, b));
    }
    const int m = min(n - at, left);
    const Run r = run_of(A, b);
    Sums<T, HD, NT> W;
    walk<T, HD, NT>(A, W, r, b, g, 0, at * kGrain, (at + m) * kGrain, r.C, r.L - 1, wave,
                        lane);
    finish<T, HD, NT>(A, W, r, g, 0, m == n ? -1 : 2 * (long)w + !start, s_o, s_m, wave,
                          lane);
    at += m, left -= m;
  }
  for (int e = w; e < A.P.B; e += A.wgs) {
    const Run r = run_of(A, e);
    if (r.none || r.nan)
      for (int g = 0; g < nkv; ++g) fill<T, HD>(A, r, g, 0, 1);
  }
  for (int g = 0; g < nkv; ++g) fill_rest<T, HD>(A, g, w, A.wgs);
}

// The entries of a head whose positions several workgroups had, joined: a workgroup per
// row, HD / 4 lanes across and 256 / (HD / 4) entries at a time.
template <class T, int HD>
__global__ __launch_bounds__(256) void join_kernel(Attend<T> A) {
  constexpr int kAcross = HD / 4, kAt = 256 / kAcross;
  __shared__ float4v s_o[kAt][kAcross];
  __shared__ float s_m[kAt], s_l[kAt];
  const int b = blockIdx.z, g = blockIdx.y, row = blockIdx.x, nkv = A.P.nkv;
  const Run r = run_of(A, b);
  if (r.L == 0 || row >= A.rep * r.n) return;
  int below = 0, total = 0;  // grains of one head
  for (int e = threadIdx.x & 63; e < A.P.B; e += 64) {
    const int t = grains_of(A, e);
    total += t, below += e < b ? t : 0;
  }
  below = __builtin_amdgcn_readlane(lane_scan(below), 63);
  total = __builtin_amdgcn_readlane(lane_scan(total), 63);
  const int n = (r.L + kGrain - 1) / kGrain;
  const Deal D(total * nkv, A.wgs);
  const int x0 = below * nkv + g * n;  // this head's first grain
  const int w0 = D.owner(x0), w1 = D.owner(x0 + n - 1);
  if (w0 == w1) return;
  const int c = threadIdx.x % kAcross, at = threadIdx.x / kAcross;
  float m = -__builtin_inff(), sum = 0.f;
  float4v o = (float4v)(0.f);
  const float* ms = A.part + 2 * (long)A.wgs * A.R * HD;
  for (int w = w0 + at; w <= w1; w += 4 * kAt) {
    float em[4], el[4];
    float4v eo[4];  // four entries asked for together
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int x = min(w + i * kAt, w1);
      const long e = (2 * (long)x + (D.from(x) < x0)) * A.R + row;
      em[i] = ms[2 * e], el[i] = ms[2 * e + 1];
      eo[i] = *reinterpret_cast<const float4v*>(A.part + e * HD + 4 * c);
    }
    float nm = m;
#pragma unroll
    for (int i = 0; i < 4; ++i) nm = fmaxf(nm, em[i]);
    const float ref = nm == -__builtin_inff() ? 0.f : nm;
    const float a = weight(m - ref);
    o *= a, sum *= a, m = nm;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (w + i * kAt > w1) continue;
      const float z = weight(em[i] - ref);
      o += eo[i] * z, sum += el[i] * z;
    }
  }
  s_o[at][c] = o;
  if (c == 0) s_m[at] = m, s_l[at] = sum;
  __syncthreads();
  if (at) return;
#pragma unroll
  for (int i = 0; i < kAt; ++i) m = fmaxf(m, s_m[i]);
  const float ref = m == -__builtin_inff() ? 0.f : m;
  o = (float4v)(0.f), sum = 0.f;
#pragma unroll
  for (int i = 0; i < kAt; ++i) {
    const float a = weight(s_m[i] - ref);
    o += s_o[i][c] * a, sum += s_l[i] * a;
  }
  const int tok = row / A.rep, head = row - tok * A.rep;
  T* dst = A.out + (long)(r.row + tok) * A.ld_o + (long)(g * A.rep + head) * HD + 4 * c;
  const float is = 1.f / sum;
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = (T)(o[i] * is);
}

// Pages src[i] to dst[i] of every layer; the addresses and pairs go in the arguments.  (64
// pages of 32 layers, 8 heads of 128 and 64 positions, 215 us, 5.0 TB/s; one page 11.6.)
constexpr int kLayers = 64, kPairs = 64;
struct Copies {
  void *k[kLayers], *v[kLayers];
  int src[kPairs], dst[kPairs];
};
__global__ __launch_bounds__(256) void copy_kernel(Copies c, long vecs) {
  u32x4* base = reinterpret_cast<u32x4*>(blockIdx.z ? c.v[blockIdx.y] : c.k[blockIdx.y]);
  const u32x4* from = base + c.src[blockIdx.x] * vecs;
  u32x4* to = base + c.dst[blockIdx.x] * vecs;
  for (long i = threadIdx.x; i < vecs; i += 256) to[i] = from[i];
}

bool fits(long hd, long page) {
  return (hd == 64 || hd == 128 || hd == 256) && page >= 16 && page <= 1024 &&
         (page & (page - 1)) == 0;
}

bool heads_fit(const hn_paged_step* s) {
  return s->nkv > 0 && s->nh > 0 && s->nh % s->nkv == 0 && s->nh < 1 << 16;
}

// Whether the attention's launches hold the rows of a sequence.  (The heads fit.)
bool rows_fit(const hn_paged_step* s) {
  return s->max_new >= 1 && s->bound >= 1 && s->max_new <= (1l << 24) / s->nh &&
         s->nh / s->nkv * s->max_new <= 65535l * kBlock;
}

// Checks a step, and fills what the kernels take of it.
int check_step(const char* who, const hn_paged_step* s, const void* x, const void* k,
               const void* v, int dtype, Step& P) {
  HN_ARG_CHECK(s, "%s: null step", who);
  HN_ARG_CHECK(dtype == 0 || dtype == 1, "%s: dtype %d (0 fp16, 1 bf16)", who, dtype);
  HN_ARG_CHECK(heads_fit(s), "%s: %ld heads over %ld KV heads", who, s->nh, s->nkv);
  HN_ARG_CHECK(fits(s->hd, s->page), "%s: heads of 64, 128 or 256 (got %ld), pages of 16 to 1024 "
               "positions, a power of two (got %ld)", who, s->hd, s->page);
  HN_ARG_CHECK(s->B >= 0 && s->B < 65536 && s->T >= 0 && s->T < 1 << 30 && s->num_pages >= 0 &&
                   s->cols >= 0 && s->ld_table >= s->cols && (s->starts || s->T == s->B),
               "%s: %ld sequences, %ld rows, %ld pages, a table of %ld columns (row %ld)", who,
               s->B, s->T, s->num_pages, s->cols, s->ld_table);
  P = Step{s->table, s->ld_table, s->cols, s->num_pages, s->lens, s->starts, (int)s->B, (int)s->T,
           (int)s->nkv, (int)s->page};
  if (s->B == 0 || s->T == 0) return 0;
  HN_ARG_CHECK(x && k && v && (s->cols == 0 || s->table) && s->lens, "%s: null operand", who);
  HN_ARG_CHECK(((uintptr_t)k | (uintptr_t)v) % 16 == 0, "%s: pages not 16-byte aligned", who);
  return 0;
}

// Rows from which a thread takes four heads of a token, so that it reads the angles once
// (8928 rows 54 us, with one head a thread 77; 500 7.3 / 8.1, 100 5.2 / 5.2, 64 single tokens
// 5.7 / 5.0).
constexpr int kManyRows = 256;

template <class T, int HD>
void append_rows(const Step& P, const T* qkv, long ld, const float* cos_t, const float* sin_t,
                 long rows, int rd, int pairs, int nh, T* q_out, T* k, T* v, hipStream_t stream) {
  constexpr int kSlots = 256 / (HD / 16);
  const bool many = P.T >= kManyRows;
  const int across = many ? 1 : kSlots, heads = many ? 4 : kSlots;
  const int qy = hn_cdiv(nh + P.nkv, heads), qk = qy * hn_cdiv(P.T, kSlots / across);
  const long groups = P.starts ? hn_cdiv(P.T, 8) : P.T;
  const int grid = qk + hn_cdiv(groups * P.nkv * (HD / 8), 256);
  if (many)
    append_rows_kernel<T, HD, 4><<<grid, 256, 0, stream>>>(
        P, qkv, ld, cos_t, sin_t, rows, rd, pairs, nh, across, qy, qk, q_out, k, v);
  else
    append_rows_kernel<T, HD, 1><<<grid, 256, 0, stream>>>(
        P, qkv, ld, cos_t, sin_t, rows, rd, pairs, nh, across, qy, qk, q_out, k, v);
}

template <class T>
int append(const Step& P, const void* qkv_, long ld, const float* cos_t, const float* sin_t,
           long rows, int rd, int pairs, int nh, int hd, void* q_, void* k_, void* v_,
           hipStream_t stream) {
  const T* qkv = (const T*)qkv_;
  T *q = (T*)q_, *k = (T*)k_, *v = (T*)v_;
  const bool vectors = ((uintptr_t)qkv | (uintptr_t)q | (uintptr_t)cos_t | (uintptr_t)sin_t) % 16 == 0 &&
                       ld % 8 == 0 && rd % 16 == 0;
  if (!vectors)
    append_kernel<T><<<dim3(P.T, nh + 2 * P.nkv), hd, 0, stream>>>(P, qkv, ld, cos_t, sin_t, rows,
                                                                  rd, pairs, nh, hd, q, k, v);
  else if (hd == 64) append_rows<T, 64>(P, qkv, ld, cos_t, sin_t, rows, rd, pairs, nh, q, k, v, stream);
  else if (hd == 128) append_rows<T, 128>(P, qkv, ld, cos_t, sin_t, rows, rd, pairs, nh, q, k, v, stream);
  else append_rows<T, 256>(P, qkv, ld, cos_t, sin_t, rows, rd, pairs, nh, q, k, v, stream);
  HN_LAUNCH_CHECK("hn_paged_append");
  return 0;
}

// Rows of one (sequence, KV head) up to which a workgroup takes all of them for a share of
// the positions, as many as its waves' registers hold; more go by blocks.  (Shared / by
// blocks, us, 8 KV heads of 128: 20 rows of 1 sequence of 3000 13.0 / 17.4, of 8 28.2 / 33.4, of
// 64 149 / 163; 32 rows 15.3 / 18.0, 30.9 / 32.5, 156 / 164, of 64 of 150 to 8000 230 / 322.)
constexpr int share_rows(long hd) { return hd == 256 ? 16 : 32; }

// How a call runs, by its sizes alone: wgs workgroups that share the positions, or, with 0,
// one per head; of runs of many rows, one per block and share of its positions, of `each`
// stages.
struct Way {
  bool blocks;
  int wgs, shares, each;
  long entries, bytes;  // of workspace
};

// One per head needs no join, but its longest head is the last to end, and few heads leave
// the chip idle.  (One token, 8 KV heads of 128, shared / per head, us: 1 sequence of 100 8.5
// / 5.8, of 300 9.2 / 11.9, of 700 9.9 / 17; 64 of 250 22.9 / 18.4, of 1000 54 / 49, of 150 to
// 8000 200 / 241; 256 of 1 to 1000 138 / 107.)
Way way_of(long B, long nh, long nkv, long hd, long max_new, long bound) {
  const long rows = nh / nkv * max_new, heads = B * nkv;
  bound = min(bound, 1l << 30);  // (no table has more positions)
  const int cus = hn_device_cus(), wgs = cus * resident(hd);
  Way x = {rows > share_rows(hd), 0, 1, 1 << 30, 0, 0};
  if (x.blocks) {
    const long blocks = heads * hn_cdiv(rows, kBlock);
    x.shares = (int)max(1l, min(wgs / blocks, bound / kShare));
    if (x.shares > 1) {
      x.each = hn_cdiv(hn_cdiv(bound, stage_of(hd)), x.shares);
      x.entries = blocks * x.shares;
      x.bytes = x.entries * kBlock * (hd + 2) * 4;
    }
  } else {
    x.wgs = bound <= kGrain || (heads >= 2 * cus && bound <= 1024 * (heads / cus)) ? 0 : wgs;
    x.bytes = 2l * x.wgs * rows * (hd + 2) * 4;
  }
  return x;
}

template <class T, int HD, int NT>
int attend_rows(const Attend<T>& A, int B, int nkv, hipStream_t stream) {
  if (A.wgs) {
    share_kernel<T, HD, NT><<<A.wgs, 256, 0, stream>>>(A);
    HN_LAUNCH_CHECK("hn_paged_attention");
    join_kernel<T, HD><<<dim3(A.R, nkv, B), 256, 0, stream>>>(A);
  } else {
    whole_kernel<T, HD, NT>
        <<<dim3(nkv, hn_cdiv(A.R, 16 * NT), B), 64 * NW, 0, stream>>>(A);
  }
  HN_LAUNCH_CHECK("hn_paged_attention");
  return 0;
}

template <class T, int HD>
int attend_hd(const Attend<T>& A, bool by_blocks, int B, int nkv, hipStream_t stream) {
  if (by_blocks) {
    const int blocks = hn_cdiv(A.R, kBlock);
    block_kernel<T, HD><<<dim3(nkv, blocks * A.shares, B), 256, 0, stream>>>(A);
    HN_LAUNCH_CHECK("hn_paged_attention");
    if (A.shares == 1) return 0;
    join_blocks_kernel<T, HD><<<dim3(nkv, blocks * (HD / 8), B), 256, 0, stream>>>(A);
    HN_LAUNCH_CHECK("hn_paged_attention");
    return 0;
  }
  if (A.R <= 16) return attend_rows<T, HD, 1>(A, B, nkv, stream);
  return attend_rows<T, HD, HD == 256 ? 1 : 2>(A, B, nkv, stream);
}

template <class T>
int attend(const Step& P, const void* q, long ld_q, const void* k, const void* v, int nh, int hd,
           int max_new, const Way& way, float scale, void* out, long ld_o, void* work,
           hipStream_t stream) {
  const int rep = nh / P.nkv;
  const Attend<T> A = {P, (const T*)q, (const T*)k, (const T*)v, (T*)out, (float*)work, ld_q, ld_o,
                       rep, max_new, rep * max_new, way.wgs, way.shares, way.each, way.entries,
                       scale};
  if (hd == 64) return attend_hd<T, 64>(A, way.blocks, P.B, P.nkv, stream);
  if (hd == 128) return attend_hd<T, 128>(A, way.blocks, P.B, P.nkv, stream);
  return attend_hd<T, 256>(A, way.blocks, P.B, P.nkv, stream);
}

}  // namespace

extern "C" int hn_paged_append(const hn_paged_step* step, const void* qkv, long ld_qkv, int dtype,
                               const float* cos_t, const float* sin_t, long table_rows,
                               long rotary, int interleaved, void* q_out, void* k, void* v,
                               void* stream) {
  Step P;
  if (int rc = check_step("hn_paged_append", step, qkv, k, v, dtype, P)) return rc;
  const long nh = step->nh, hd = step->hd, heads = nh + 2 * step->nkv;
  HN_ARG_CHECK(rotary >= 0 && rotary <= hd && rotary % 2 == 0 && table_rows >= 0,
               "hn_paged_append: %ld rotated dimensions of %ld, %ld positions", rotary, hd,
               table_rows);
  HN_ARG_CHECK(heads < 65536 && P.T * heads < 1l << 31, "hn_paged_append: %d rows of %ld heads",
               P.T, heads);
  if (P.B == 0 || P.T == 0) return 0;
  HN_ARG_CHECK(q_out && (rotary == 0 || (cos_t && sin_t)), "hn_paged_append: null operand");
  HN_ARG_CHECK(ld_qkv >= heads * hd, "hn_paged_append: rows of %ld, a stride of %ld", heads * hd,
               ld_qkv);
  return (dtype == 0 ? append<h16> : append<b16>)(P, qkv, ld_qkv, cos_t, sin_t, table_rows,
                                                  (int)rotary, interleaved, (int)nh, (int)hd,
                                                  q_out, k, v, (hipStream_t)stream);
}

extern "C" long hn_paged_attention_workspace_bytes(const hn_paged_step* s) {
  // (0 too for what the call refuses)
  if (!s || s->B <= 0 || s->B >= 65536 || s->T <= 0 || !heads_fit(s) || !fits(s->hd, s->page) ||
      !rows_fit(s))
    return 0;
  return way_of(s->B, s->nh, s->nkv, s->hd, s->max_new, s->bound).bytes;
}

extern "C" int hn_paged_attention(const hn_paged_step* step, const void* q, long ld_q, int dtype,
                                  const void* k, const void* v, float scale, void* out, long ld_o,
                                  void* work, long work_bytes, void* stream) {
  Step P;
  if (int rc = check_step("hn_paged_attention", step, q, k, v, dtype, P)) return rc;
  const long nh = step->nh, nkv = step->nkv, hd = step->hd, max_new = step->max_new;
  HN_ARG_CHECK(rows_fit(step), "hn_paged_attention: max_new %ld, bound %ld", max_new,
               step->bound);
  HN_ARG_CHECK(P.cols < 1l << 26 && P.cols * P.page < 1l << 30 &&
                   (double)P.B * nkv * (P.cols * P.page / kGrain + 1) < 2147483648.0,
               "hn_paged_attention: %d sequences of %ld pages", P.B, P.cols);
  HN_ARG_CHECK(scale > 0.f && scale * 1.4426950408889634f < __builtin_inff(),
               "hn_paged_attention: scale %g", (double)scale);
  if (P.B == 0 || P.T == 0) return 0;
  HN_ARG_CHECK(P.pages >= 1, "hn_paged_attention: no pages");
  HN_ARG_CHECK(out && ld_q >= nh * hd && ld_o >= nh * hd && ld_q % 8 == 0 && ld_o % 8 == 0 &&
                   ((uintptr_t)q | (uintptr_t)out) % 16 == 0,
               "hn_paged_attention: rows of %ld, strides of %ld and %ld: 16-byte aligned rows",
               nh * hd, ld_q, ld_o);
  const Way way = way_of(P.B, nh, nkv, hd, max_new, step->bound);
  HN_ARG_CHECK(way.bytes == 0 || (work && (uintptr_t)work % 16 == 0 && work_bytes >= way.bytes),
               "hn_paged_attention: a workspace of %ld bytes, %ld given", way.bytes,
               work ? work_bytes : 0);
  return (dtype == 0 ? attend<h16> : attend<b16>)(P, q, ld_q, k, v, (int)nh, (int)hd,
                                                  (int)max_new, way, scale, out, ld_o, work,
                                                  (hipStream_t)stream);
}

extern "C" int hn_page_copy(void* const* k, void* const* v, long layers, long page_bytes,
                            long num_pages, const int* src, const int* dst, long pairs,
                            void* stream) {
  HN_ARG_CHECK(layers >= 0 && pairs >= 0 && page_bytes > 0 && page_bytes % 16 == 0,
               "hn_page_copy: %ld layers, %ld pairs, pages of %ld bytes", layers, pairs,
               page_bytes);
  if (layers == 0 || pairs == 0) return 0;
  HN_ARG_CHECK(k && v && src && dst, "hn_page_copy: null operand");
  for (long i = 0; i < pairs; ++i)
    HN_ARG_CHECK(src[i] >= 0 && src[i] < num_pages && dst[i] >= 0 && dst[i] < num_pages,
                 "hn_page_copy: page %d to %d of %ld", src[i], dst[i], num_pages);
  for (long l = 0; l < layers; ++l)
    HN_ARG_CHECK(k[l] && v[l] && ((uintptr_t)k[l] | (uintptr_t)v[l]) % 16 == 0,
                 "hn_page_copy: layer %ld: a null or unaligned address", l);
  for (long l0 = 0; l0 < layers; l0 += kLayers)
    for (long p0 = 0; p0 < pairs; p0 += kPairs) {
      Copies c = {};
      const int nl = (int)(layers - l0 < kLayers ? layers - l0 : kLayers);
      const int np = (int)(pairs - p0 < kPairs ? pairs - p0 : kPairs);
      for (int l = 0; l < nl; ++l) c.k[l] = k[l0 + l], c.v[l] = v[l0 + l];
      for (int i = 0; i < np; ++i) c.src[i] = src[p0 + i], c.dst[i] = dst[p0 + i];
      copy_kernel<<<dim3(np, nl, 2), 256, 0, (hipStream_t)stream>>>(c, page_bytes / 16);
      HN_LAUNCH_CHECK("hn_page_copy");
    }
  return 0;
}
