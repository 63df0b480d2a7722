// Attention of a tree of drafted tokens over the KV cache: the plan of a tree,
// RoPE and the cache append of its nodes, and the attention.
//
// A tree is a row of parents, node i below parents[i] < i (-1: directly below
// the cached positions).  A node with any other parent, and every node below
// it, is padding.  Node i of a sequence with C = lens[b] cached positions sits
// at cache position C + i, its rotary position is C + depth(i), and it sees
// positions [0, C) and those of itself and its ancestors.
#include <float.h>

#include "hn_common.h"
#include "hn_lds_dma.h"

namespace {

constexpr int kHd = 128;
constexpr int kMaxNodes = 256;
constexpr int kWords = kMaxNodes / 64;
typedef unsigned long long u64;

// One workgroup per tree, a thread per node.  Pointer doubling: after round r a
// node has joined the sets of 2^r ancestors and points 2^r above itself, so a
// chain of 256 takes 8 rounds.  A padding node points at itself with no set; a
// node that meets one on its way becomes padding too.
__global__ __launch_bounds__(kMaxNodes) void plan_kernel(const int* __restrict__ parents, long ld_p,
                                                         int S, int* __restrict__ up,
                                                         int* __restrict__ depth,
                                                         u64* __restrict__ seen) {
  __shared__ u64 set[kMaxNodes][kWords];
  __shared__ int ptr[kMaxNodes];  // -1: past the root, -2: padding
  const int b = blockIdx.x, i = threadIdx.x;
  const int p = i < S ? parents[(long)b * ld_p + i] : -2;
  const int mine = i < S && p >= -1 && p < i ? p : -2;
  ptr[i] = mine;
#pragma unroll
  for (int w = 0; w < kWords; ++w) set[i][w] = w == i >> 6 ? 1ull << (i & 63) : 0ull;
  __syncthreads();
  for (int step = 1; step < S; step <<= 1) {
    u64 s[kWords];
    const int at = ptr[i];
    int to = at;
    if (at >= 0) {
      to = ptr[at];
#pragma unroll
      for (int w = 0; w < kWords; ++w) s[w] = set[i][w] | set[at][w];
    }
    __syncthreads();
    if (at >= 0) {
      ptr[i] = to;
#pragma unroll
      for (int w = 0; w < kWords; ++w) set[i][w] = s[w];
    }
    __syncthreads();
  }
  if (i >= S) return;
  const bool live = ptr[i] == -1;
  const long o = (long)b * S + i;
  int n = -1;
#pragma unroll
  for (int w = 0; w < kWords; ++w) {
    const u64 s = live ? set[i][w] : 0ull;
    n += __popcll(s);
    seen[o * kWords + w] = s;
  }
  up[o] = live ? mine : -2;
  depth[o] = n;
}

// Where a node goes.  in: its position is in the table and the cache; live: it
// takes part.
struct Place {
  long pos, slot;
  bool live, in;
};
__device__ __forceinline__ Place place(const int* depth, int trees, const long* lens, int b, int i,
                                       int S, long table_rows, long max_len) {
  const int dep = depth[(trees > 1 ? (long)b * S : 0) + i];
  const long C = lens[b];
  Place p = {0, 0, C >= 0 && dep >= 0, false};
  p.in = p.live && C < table_rows - dep && C < max_len - i;
  if (p.in) p.pos = C + dep, p.slot = C + i;
  return p;
}

// A thread per element of a head, grid (B * S, nh + nkv): rows of any alignment.
__global__ __launch_bounds__(kHd) void append_kernel(
    const h16* __restrict__ qkv, long ld, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, long table_rows, const int* __restrict__ depth, int trees,
    const long* __restrict__ lens, int S, int nkv, int rep, h16* __restrict__ q_out,
    h16* __restrict__ kt, h16* __restrict__ vc, long max_len) {
  const int row = blockIdx.x, head = blockIdx.y, d = threadIdx.x;
  const int b = row / S, i = row - b * S, nh = nkv * rep;
  const Place at = place(depth, trees, lens, b, i, S, table_rows, max_len);
  const long pos = at.pos, slot = at.slot;
  const bool live = at.live, in = at.in;
  const h16* src = qkv + (long)row * ld + (long)head * kHd;
  float y = 0.f;
  if (in) {
    const float x = (float)src[d], z = (float)src[d ^ (kHd / 2)];
    y = x * cos_t[pos * kHd + d] + (d < kHd / 2 ? -z : z) * sin_t[pos * kHd + d];
  } else if (live) {
    y = __builtin_nanf("");
  }
  if (head < nh) {
    const int g = head / rep, r = head - g * rep;
    q_out[((((long)b * nkv + g) * rep + r) * S + i) * kHd + d] = (h16)y;
  } else if (in) {
    const int g = head - nh;
    kt[(((long)b * nkv + g) * kHd + d) * max_len + slot] = (h16)y;
    vc[(((long)b * nkv + g) * max_len + slot) * kHd + d] = src[(long)nkv * kHd + d];
  }
}

// The same for 16-byte aligned rows: 32 nodes per workgroup, 8 lanes each, a lane
// 8 elements of a head's lower half and their partners of the upper, so every
// access of q, k and v is 16 bytes and the angles stay in registers over the
// heads.  The rotated keys go through LDS, to be written with lanes along the
// nodes, whose positions are consecutive.  Grid (ceil(B S / 32), ceil(nh / 4) +
// nkv): groups of query heads, then a KV head each.
constexpr int kAppend = 32, kHeads = 4, kKPad = kAppend + 2;
typedef float float8v __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void rotate8(half8_t x, half8_t y, float8v cl, float8v ch, float8v sl,
                                        float8v sh, half8_t& lo, half8_t& hi) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = (h16)((float)x[e] * cl[e] - (float)y[e] * sl[e]);
    hi[e] = (h16)((float)y[e] * ch[e] + (float)x[e] * sh[e]);
  }
}

__global__ __launch_bounds__(256) void append_rows_kernel(
    const h16* __restrict__ qkv, long ld, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, long table_rows, const int* __restrict__ depth, int trees,
    const long* __restrict__ lens, int B, int S, int nkv, int rep, h16* __restrict__ q_out,
    h16* __restrict__ kt, h16* __restrict__ vc, long max_len) {
  constexpr int half = kHd / 2;
  __shared__ h16 s_k[kHd * kKPad];
  const int tid = threadIdx.x, tok = tid >> 3, d = 8 * (tid & 7), nh = nkv * rep;
  const int row = blockIdx.x * kAppend + tok;
  const bool there = row < B * S;
  const int b = there ? row / S : 0, i = there ? row - b * S : 0;
  const Place at = place(depth, trees, lens, b, i, S, table_rows, max_len);
  const bool live = at.live && there, in = at.in && there;
  float8v cl, ch, sl, sh;
  if (in) {
    const float* c = cos_t + at.pos * kHd + d;
    const float* s = sin_t + at.pos * kHd + d;
    cl = *reinterpret_cast<const float8v*>(c), ch = *reinterpret_cast<const float8v*>(c + half);
    sl = *reinterpret_cast<const float8v*>(s), sh = *reinterpret_cast<const float8v*>(s + half);
  }
  const h16* src = qkv + (long)row * ld;
  const int groups = (nh + kHeads - 1) / kHeads;
  if ((int)blockIdx.y < groups) {
    if (!there) return;
    const int h0 = blockIdx.y * kHeads;
    half8_t x[kHeads], y[kHeads];  // all loads before the first store
    if (in)
#pragma unroll
      for (int k = 0; k < kHeads; ++k) {
        const h16* p = src + (long)(h0 + k < nh ? h0 + k : nh - 1) * kHd + d;
        x[k] = *reinterpret_cast<const half8_t*>(p);
        y[k] = *reinterpret_cast<const half8_t*>(p + half);
      }
    // zero for padding, NaN past the cache or the table
    const h16 none = live ? (h16)__builtin_nanf("") : (h16)0.f;
#pragma unroll
    for (int k = 0; k < kHeads; ++k) {
      half8_t lo, hi;
#pragma unroll
      for (int e = 0; e < 8; ++e) lo[e] = hi[e] = none;
      if (in) rotate8(x[k], y[k], cl, ch, sl, sh, lo, hi);
      if (h0 + k < nh) {
        h16* dst = q_out + (((long)b * nh + h0 + k) * S + i) * kHd + d;
        *reinterpret_cast<half8_t*>(dst) = lo;
        *reinterpret_cast<half8_t*>(dst + half) = hi;
      }
    }
    return;
  }
  const int g = blockIdx.y - groups;
  if (in) {
    const h16* ks = src + (long)(nh + g) * kHd + d;
    const h16* vs = src + (long)(nh + nkv + g) * kHd + d;
    const half8_t x = *reinterpret_cast<const half8_t*>(ks);
    const half8_t y = *reinterpret_cast<const half8_t*>(ks + half);
    const half8_t v0 = *reinterpret_cast<const half8_t*>(vs);
    const half8_t v1 = *reinterpret_cast<const half8_t*>(vs + half);
    h16* vd = vc + (((long)b * nkv + g) * max_len + at.slot) * kHd + d;
    *reinterpret_cast<half8_t*>(vd) = v0;
    *reinterpret_cast<half8_t*>(vd + half) = v1;
    half8_t lo, hi;
    rotate8(x, y, cl, ch, sl, sh, lo, hi);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s_k[(d + e) * kKPad + tok] = lo[e];
      s_k[(d + half + e) * kKPad + tok] = hi[e];
    }
  }
  __syncthreads();
  const int r2 = blockIdx.x * kAppend + (tid & (kAppend - 1));
  if (r2 >= B * S) return;
  const int b2 = r2 / S, i2 = r2 - b2 * S;
  const Place to = place(depth, trees, lens, b2, i2, S, table_rows, max_len);
  if (!to.in) return;
  h16* kd = kt + ((long)b2 * nkv + g) * kHd * max_len + to.slot;
#pragma unroll
  for (int e = 0; e < kHd / 8; ++e) {
    const int dd = 8 * e + (tid >> 5);
    kd[(long)dd * max_len] = s_k[dd * kKPad + (tid & (kAppend - 1))];
  }
}

// ---------------------------------------------------------------------------
// Attention.  One pass over the cache with a running maximum and sum, for the rows
// of one (sequence, KV head), a row being a (query head of the group, node) pair:
//   S^T = K Q^T    v_mfma_f32_16x16x32_f16, A = K, B = Q;
//   softmax        a lane holds scores of one row;
//   O^T += V^T P   the lane's probabilities are the B operand as they are.
// share_kernel walks the positions, join_kernel adds up what several workgroups
// made of one head.
//
// Bounds, and time where the workgroups hold 8 KV heads of 128 and 4 query heads
// each (a large copy moves 4.9 TB/s):
//   32 sequences of 8000, 4 nodes     the cache's bytes: 222 us, 4.7 TB/s
//   1 of 30000, 4 nodes               37 us, 3.3 TB/s
//   8 of 8000, 64 nodes               120 us, 0.58 PFLOP/s: the softmax and the
//                                     LDS reads between the products
//   1 of 300, 1 node                  13 us: two launches, and memory's latency
// Positions that workgroups share out as one.  Of 64 a head's ranges need not start
// on 256 bytes of its keys: 245 us for the first of the cases above, 222 of 128.
constexpr int kGrain = 128;
constexpr int kOPad = kHd + 4;
constexpr uint32_t kNone = 0xfffff000u;  // an offset past any descriptor: reads zero, no access
constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are 2^8 times the softmax's, relative to a maximum that follows
// the true one only when it lags by 2^6: below 2^14, so fp16 holds them, and
// those down to 2^-22 of the largest are normal numbers.  They are rounded to fp16
// because that is what the matrix instruction multiplies with fp16 values (in two
// parts, high and low, the second product would take twice as many); a row's sum is
// of the rounded ones, so that their weights still add up to 1.  The rows' relative
// error against 64 bits is 2.3e-4 to 2.7e-4 in the cases above, of which rounding
// the result to fp16 alone is 2.1e-4.
constexpr float kUp = 8.f, kLag = 6.f;

typedef float float4v __attribute__((ext_vector_type(4)));

template <bool B>
struct Bool {
  static constexpr bool value = B;
};

struct Attend {
  const h16 *q, *kt, *v;
  const long* lens;
  const u64* seen;
  h16* out;
  float* part;
  long max_len, bound, ld_o;
  int trees, B, nkv, rep, S, R, blocks, wgs;
  float scale;
};

// max over the four lanes, 16 apart, that hold one row.  (The swapped pair goes
// through scalars: a bit cast of a vector's element takes element 0.)
__device__ __forceinline__ float row_max(float x) {
  const uint32_t w = __builtin_bit_cast(uint32_t, x);
  const auto a = __builtin_amdgcn_permlane16_swap(w, w, false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  x = fmaxf(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  const uint32_t v = __builtin_bit_cast(uint32_t, x);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return fmaxf(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

// Bits [at, at + 32) of what a node sees, positions before its tree (at < 0) all
// seen.
__device__ __forceinline__ uint32_t window(const u64* see, int at) {
  if (at <= -32) return ~0u;
  if (at >= kMaxNodes) return 0u;
  if (at < 0) return (uint32_t)(see[0] << -at) | ((1u << -at) - 1u);
  const int w = at >> 6, s = at & 63;
  u64 x = see[w] >> s;
  if (s > 32 && w + 1 < kWords) x |= see[w + 1] << (64 - s);
  return (uint32_t)x;
}

// The halves of w that are NaN or infinite, as a mask.
__device__ __forceinline__ uint32_t odd_mask(uint32_t w) {
  return ((w & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) |
         ((w & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}

// The work is cut into grains of kGrain positions of one (sequence, KV head), in
// order, and each workgroup takes as many of them as the others (or one less),
// whatever the sequences' lengths, which only the device knows.  Such a share is
// one range of positions of one head or several; a head's range that is not whole
// leaves its sums in the workspace, in entry 2 w of workgroup w, or 2 w + 1 if it
// is not w's first, for join_kernel.  The row blocks of a share follow each other
// on one XCD, whose L2 then serves all but the first.
__device__ __forceinline__ int grains_of(const Attend& A, int b) {
  const long C = A.lens[b];
  return C < 0 || C > A.bound - A.S ? 0 : ((int)C + A.S + kGrain - 1) / kGrain;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

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

// Grains of one head of the sequences below `to`, by a wave.
__device__ __forceinline__ int grains_below(const Attend& A, int to) {
  int n = 0;
  for (int b = threadIdx.x & 63; b < to; b += 64) n += grains_of(A, b);
  return __builtin_amdgcn_readlane(lane_scan(n), 63);
}

// T grains over the workgroups: the first `more` take each + 1 of them.
struct Split {
  int wgs, each, more;
  __device__ Split(int T, int most) : wgs(T < most ? T : most) {
    each = wgs ? (int)((unsigned)T / (unsigned)wgs) : 0, more = T - each * wgs;
  }
  __device__ int from(int w) const { return w * each + (w < more ? w : more); }
  __device__ int owner(int x) const {
    const int big = more * (each + 1);
    return x < big ? (int)((unsigned)x / (unsigned)(each + 1))
                   : more + (int)((unsigned)(x - big) / (unsigned)each);
  }
};

// A range of positions of one KV head: grains [first, end).
struct Where {
  int bg, b, g, row0, tree, first, end;
  int C, L;     // cached positions, and with the nodes
  bool whole;   // all of the head's
  long part;    // else its entry of the workspace
};

struct Share {
  int w, block, b, g, at, n;  // next: grain `at` of the n of head g of sequence b
  int left;                   // grains left
  bool first;

  __device__ bool begin(const Attend& A) {
    const int id = blockIdx.x, grp = id / (8 * A.blocks), in = id - grp * 8 * A.blocks;
    w = 8 * grp + (in & 7), block = in >> 3;
    if (w >= A.wgs) return false;
    const Split P(grains_below(A, A.B) * A.nkv, A.wgs);
    first = true, b = 0, g = 0, at = 0, n = 0, left = 0;
    if (w >= P.wgs) return true;
    const int from = P.from(w);
    left = P.from(w + 1) - from;
    const int lane = threadIdx.x & 63;
    int base = 0;  // grains of one head of the sequences before
    for (int c = 0; c < A.B; c += 64) {
      const int t = c + lane < A.B ? grains_of(A, c + lane) : 0;
      const int sum = lane_scan(t);
      const u64 past = __ballot((base + sum) * A.nkv > from);
      if (past) {
        const int l = __builtin_ctzll(past);
        b = c + l;
        n = __builtin_amdgcn_readlane(t, l);
        const int in_b = from - (base + __builtin_amdgcn_readlane(sum, l) - n) * A.nkv;
        g = (int)((unsigned)in_b / (unsigned)n), at = in_b - g * n;
        break;
      }
      base += __builtin_amdgcn_readlane(sum, 63);
    }
    return true;
  }

  __device__ bool next(const Attend& A, int rows, Where& W) {
    if (left <= 0) return false;
    while (at >= n) {  // the next head that has grains
      at = 0;
      if (n > 0 && ++g < A.nkv) break;
      g = 0;
      n = uniform(grains_of(A, ++b));
    }
    const int m = n - at < left ? n - at : left;
    W.b = b, W.g = g, W.bg = b * A.nkv + g, W.row0 = block * rows;
    W.tree = A.trees > 1 ? b : 0;
    W.C = uniform((int)A.lens[b]), W.L = W.C + A.S;
    W.first = at, W.end = at + m;
    W.whole = m == n;
    W.part = 2 * (long)w + !first;
    at += m, left -= m, first = false;
    return true;
  }

  // Rows of the sequences that have no grains: zero, or NaN past the bound.
  __device__ void rest(const Attend& A, int rows) {
    for (int e = w; e < A.B; e += A.wgs) {
      if (grains_of(A, e)) continue;
      const u64* seen = A.seen + (A.trees > 1 ? (long)e * A.S : 0) * kWords;
      const int cols = A.nkv * A.rep * (kHd / 8);
      for (long i = (long)block * blockDim.x + threadIdx.x; i < (long)A.S * cols;
           i += (long)A.blocks * blockDim.x) {
        const int node = (int)(i / cols), col = (int)(i - (long)node * cols);
        const bool live =
            A.lens[e] >= 0 && ((seen[(long)node * kWords + (node >> 6)] >> (node & 63)) & 1);
        half8_t y;
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = live ? (h16)__builtin_nanf("") : (h16)0.f;
        *reinterpret_cast<half8_t*>(A.out + ((long)e * A.S + node) * A.ld_o + 8 * col) = y;
      }
    }
  }
};

// The sums of 16 rows of each of RG row groups, PG waves each, joined: wave rg *
// PG + pg has left them in s_o, s_m and s_l.  Then the rows themselves where the
// range is whole, else the range's sums.  `t`: which 16 of a
// group's `per` rows.
template <int RG, int PG>
__device__ __forceinline__ void finish(const Attend& A, const Where& W, const float* s_o,
                                       const float* s_m, const float* s_l, int t, int per) {
  for (int i = threadIdx.x; i < RG * 256; i += 64 * RG * PG) {
    const int rr = (i >> 4) & 15, w0 = (i >> 8) * PG, d = 8 * (i & 15);
    const int row = W.row0 + (i >> 8) * per + 16 * t + rr;
    if (row >= A.R) continue;
    float m = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < PG; ++w) m = fmaxf(m, s_m[(w0 + w) * per + 16 * t + rr]);
    const float ref = m == -__builtin_inff() ? 0.f : m;
    float sum = 0.f, x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = 0.f;
#pragma unroll
    for (int w = 0; w < PG; ++w) {
      // a wave without tiles has sums of zero and weight exp2(-inf) = 0
      const float al = __builtin_amdgcn_exp2f(s_m[(w0 + w) * per + 16 * t + rr] - ref);
      const float* ow = s_o + ((w0 + w) * 16 + rr) * kOPad + d;
      sum += al * s_l[(w0 + w) * per + 16 * t + rr];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] += al * ow[k];
    }
    const int head = row / A.S, node = row - head * A.S;
    if (W.whole) {
      const bool live = ((A.seen[((long)W.tree * A.S + node) * kWords + (node >> 6)] >>
                                      (node & 63)) & 1);
      const float is = 1.f / sum;
      half8_t y;
#pragma unroll
      for (int k = 0; k < 8; ++k) y[k] = live ? (h16)(x[k] * is) : (h16)0.f;
      *reinterpret_cast<half8_t*>(A.out + ((long)W.b * A.S + node) * A.ld_o +
                                  (long)(W.g * A.rep + head) * kHd + d) = y;
    } else {
      const long at = W.part * A.R + row;
      float* pm = A.part + 2 * (long)A.wgs * A.R * kHd + at * 2;
#pragma unroll
      for (int k = 0; k < 8; k += 4)
        *reinterpret_cast<float4v*>(A.part + at * kHd + d + k) =
            float4v{x[k], x[k + 1], x[k + 2], x[k + 3]};
      if ((i & 15) == 0) pm[0] = m, pm[1] = sum;
    }
  }
}

// NaN and infinities among the nodes' values, which the products leave out, added
// to the rows that see them.  hd(k, r): the element that o[t][k][r] holds.
template <int RT, typename F, typename G>
__device__ __forceinline__ void add_odd(const Attend& A, const Where& W, int row0, int n,
                                        float4v (&o)[RT][8], F hd, G mine) {
  const h16* v = A.v + ((long)W.bg * A.max_len + W.C) * kHd;
  for (int a = 0; a < A.S; ++a) {
    if (!mine(W.C + a)) continue;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int row = row0 + 16 * t + n;
      const int node = row < A.R ? row % A.S : 0;
      const bool vis = (A.seen[((long)W.tree * A.S + node) * kWords + (a >> 6)] >> (a & 63)) & 1;
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = (float)v[(long)a * kHd + hd(k, r)];
          if (vis && !(__builtin_fabsf(x) < __builtin_inff())) o[t][k][r] += x;
        }
    }
  }
}

// The walk.  4 waves, RG groups of 32 rows by PG parts of a stage of SP = 64
// positions.  K is cached as [hd][position] and V as [position][hd], so both
// products contract over the axis that is not dense in memory.  A stage of keys
// [128 hd][SP] and values [SP][128 hd] goes from memory to LDS as it lies
// (buffer_load ... lds), one stage ahead, and ds_read_b64_tr_b16 turns it on the
// way to the registers: 16 lanes read 4 rows of 16 halves, and lane i gets column
// i.  The operands' layouts are the MFMA's own: a lane's scores are positions 16 j
// + 4 kg + r of its part, of row lane % 16, and with the values' rows taken as {4
// kg + r, 16 + 4 kg + r} they are the second product's operand as they are.
// Two workgroups per CU: one's loads and barriers under the other's arithmetic.
// (Waves on positions of their own that turn 8 x 8 blocks in registers with v_perm,
// without LDS: with 16 / 32 rows per wave 16.4 / 17.4 us for 16 nodes of one
// sequence of 1500 that takes 14.4 here, 241 / 227 for the first of the cases above
// and 38 / 33 for the second.)
//
// Both transposing reads take 32 bytes of each of 16 rows; a row's 16-byte chunks
// are stored at chunk ^ (2 * key(row)), so that the 8 rows that half a wave reads
// cover the 64 banks once: the counter of bank conflicts stays at 0.
constexpr int kSP = 64;
__device__ __forceinline__ int key_of_k(int hd) { return ((hd >> 1) & 1) | ((hd >> 2) & 2); }

typedef short short4v __attribute__((ext_vector_type(4)));

// Two transposing reads: columns of 4 rows each, 8 halves of one column per lane.
__device__ __forceinline__ half8_t read_tr(uint32_t at, int lo, int hi) {
  typedef __attribute__((address_space(3))) short4v* P;
  __attribute__((address_space(3))) char* base = (__attribute__((address_space(3))) char*)nullptr + at;
  const short4v a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(base + lo));
  const short4v b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(base + hi));
  return __builtin_bit_cast(
      half8_t, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

template <int RG, int PG>
__global__ __launch_bounds__(256, 2) void share_kernel(Attend A) {
  constexpr int RT = 2, SP = kSP, WP = SP / PG, JB = WP / 16, D = 2;
  constexpr int kKBytes = SP * kHd * 2, kStage = 2 * kKBytes;
  constexpr int kDma = SP / 4 / 4;  // DMA instructions per wave and operand of a stage
  static_assert(RG * PG == 4 && D * kStage >= 4 * 16 * kOPad * 4, "");
  __shared__ __align__(1024) unsigned char s_buf[D * kStage];
  __shared__ float s_m[4 * 16 * RT], s_l[4 * 16 * RT];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, kg = lane >> 4, rg = wave / PG, pg = wave - rg * PG;
  Share share;
  if (!share.begin(A)) return;
  for (Where W; share.next(A, 32 * RG, W);) {
  const int row0 = W.row0 + 32 * rg;  // this wave's rows
  const bool busy = row0 < A.R;

  half8_t q[RT][4];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = row0 + 16 * t + n;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      u32x4 w = {0, 0, 0, 0};
      if (row < A.R)
        w = *reinterpret_cast<const u32x4*>(A.q + ((long)W.bg * A.R + row) * kHd + 32 * u + 8 * kg);
      q[t][u] = __builtin_bit_cast(half8_t, w);
    }
  }

  const long slab = (long)W.bg * kHd * A.max_len;
  const uint32_t pitch = (uint32_t)A.max_len * 2;
  const __amdgpu_buffer_rsrc_t rk = rsrc(A.kt + slab, (int)(pitch * kHd));
  const __amdgpu_buffer_rsrc_t rv = rsrc(A.v + slab, (int)(pitch * kHd));
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)s_buf;

  // DMA: instruction i of wave w moves bytes 1024 (w + 4 i) on of a stage's keys
  // and of its values; the lane's part of the addresses is the same for all i
  constexpr int kRowK = 1024 / (2 * SP), kChunks = SP / 8;  // rows of keys per instruction
  const int kr = lane / kChunks, vr = lane >> 4;
  const int kc = (lane % kChunks) ^ (2 * key_of_k(kRowK * wave + kr));
  const uint32_t kat = (uint32_t)kr * pitch + 16 * kc;
  const uint32_t vat = vr * (kHd * 2) + 16 * ((lane & 15) ^ (2 * ((4 * wave + vr) & 7)));
  const int stages = kGrain / SP * (W.end - W.first);
  // positions past the sequence read as zero: their probabilities are, and what a
  // longer sequence left there may be anything
  auto issue = [&](int st) {
    const int p0 = W.first * kGrain + st * SP;
    const uint32_t at = lds0 + (uint32_t)(st % D) * kStage + wave * 1024;
    const uint32_t ka = st < stages && p0 + 8 * kc < W.L ? kat : kNone;
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      const int qi = wave + 4 * i;
      dma_b128(rk, ka, (uint32_t)(kRowK * qi) * pitch + 2 * (uint32_t)p0, at + i * 4096);
    }
#pragma unroll
    for (int i = 0; i < kDma; ++i) {
      const int qi = wave + 4 * i;
      const uint32_t va = st < stages && p0 + 4 * qi + vr < W.L ? vat : kNone;
      dma_b128(rv, va, ((uint32_t)p0 + 4 * qi) * (kHd * 2), at + kKBytes + i * 4096);
    }
  };

  // this lane's part of the reads: 8 bytes of row (lane % 16) / 4 of a group's 4
  const int rr = n >> 2, half = 16 * ((n & 3) >> 1) + 8 * (n & 1);
  uint32_t k_at[JB], v_at[8];
#pragma unroll
  for (int j = 0; j < JB; ++j)
    k_at[j] = lds0 + (8 * kg + rr) * (2 * SP) + half +
              32 * ((pg * JB + j) ^ key_of_k(8 * kg + rr));
#pragma unroll
  for (int e = 0; e < 8; ++e)
    v_at[e] = lds0 + kKBytes + (pg * WP + 4 * kg + rr) * (kHd * 2) + half +
              32 * (e ^ ((4 * kg + rr) & 7));

  float4v o[RT][8], l[RT];
  float mx[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    mx[t] = -__builtin_inff();
    l[t] = (float4v)(0.f);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[t][e] = (float4v)(0.f);
  }
  const float scale = A.scale * kLog2e;
  half8_t ones;
#pragma unroll
  for (int i = 0; i < 8; ++i) ones[i] = (h16)1.f;
  uint32_t any_odd = 0;

  half8_t p[RT][JB / 2];
  // scores and probabilities of a stage
  auto scores = [&](auto edge_stage, int st) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge_stage)::value;
    const int p0 = W.first * kGrain + st * SP + pg * WP;
    const uint32_t at = (uint32_t)(st % D) * kStage;
    // operands are read one group of products ahead
    float4v s[RT][JB];
    half8_t ka[2][4];
    auto keys = [&](int j) {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        ka[j & 1][u] = read_tr(k_at[j] + at, u * 32 * 2 * SP, u * 32 * 2 * SP + 4 * 2 * SP);
    };
    keys(0);
#pragma unroll
    for (int j = 0; j < JB; ++j) {
      if (j + 1 < JB) keys(j + 1);
#pragma unroll
      for (int t = 0; t < RT; ++t) s[t][j] = (float4v)(0.f);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int t = 0; t < RT; ++t)
          s[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka[j & 1][u], q[t][u], s[t][j], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if constexpr (EDGE) {
        const int row = row0 + 16 * t + n;
        const int node = row < A.R ? row % A.S : 0;
        const u64* see = A.seen + ((long)W.tree * A.S + node) * kWords;
#pragma unroll
        for (int x = 0; x < JB / 2; ++x) {
          const uint32_t w = window(see, p0 + 32 * x + 4 * kg - W.C);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (!((w >> r) & 1u)) s[t][2 * x][r] = -__builtin_inff();
            if (!((w >> (16 + r)) & 1u)) s[t][2 * x + 1][r] = -__builtin_inff();
          }
        }
      }
      float tm = s[t][0][0];
#pragma unroll
      for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) tm = fmaxf(tm, s[t][j][r]);
      tm = row_max(tm) * scale;
      if (__any(tm > mx[t] + kLag)) {
        const float nm = fmaxf(mx[t], tm);
        const float al = nm == mx[t] ? 1.f : __builtin_amdgcn_exp2f(mx[t] - nm);
        l[t] *= al;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[t][e] *= al;
        mx[t] = nm;
      }
      const float ref = mx[t] == -__builtin_inff() ? 0.f : mx[t] - kUp;
#pragma unroll
      for (int j = 0; j < JB; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          p[t][j >> 1][4 * (j & 1) + r] =
              (h16)__builtin_amdgcn_exp2f(__builtin_fmaf(s[t][j][r], scale, -ref));
    }
  };
  // its values, by those probabilities
  auto values = [&](auto edge_stage, int st) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge_stage)::value;
    const int p0 = W.first * kGrain + st * SP + pg * WP;
    const uint32_t at = (uint32_t)(st % D) * kStage;
    constexpr int EB = 4;  // operands per group
    half8_t va[2][EB];
    auto read = [&](int i) {
      const int x = i * EB / 8, e0 = i * EB % 8;
#pragma unroll
      for (int e = 0; e < EB; ++e)
        va[i & 1][e] = read_tr(v_at[e0 + e] + at, x * 32 * kHd * 2, x * 32 * kHd * 2 + 16 * kHd * 2);
    };
    read(0);
#pragma unroll
    for (int i = 0; i < JB / 2 * 8 / EB; ++i) {
      const int x = i * EB / 8, e0 = i * EB % 8;
      if (i + 1 < JB / 2 * 8 / EB) read(i + 1);
      if (e0 == 0)
#pragma unroll
        for (int t = 0; t < RT; ++t)
          l[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, p[t][x], l[t], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < EB; ++e) {
        half8_t a = va[i & 1][e];
        if constexpr (EDGE) {
          // nodes' values that are no numbers: see add_odd
          u32x4 w = __builtin_bit_cast(u32x4, a);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int pos = p0 + 32 * x + 16 * (k >> 1) + 4 * kg + 2 * (k & 1);
            const uint32_t node = (pos >= W.C ? 0xffffu : 0u) | (pos + 1 >= W.C ? 0xffff0000u : 0u);
            const uint32_t m = odd_mask(w[k]) & node;
            any_odd |= m;
            w[k] &= ~m;
          }
          asm volatile("" : "+v"(any_odd));
          a = __builtin_bit_cast(half8_t, w);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
          o[t][e0 + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, p[t][x], o[t][e0 + e], 0, 0, 0);
      }
    }
  };

  issue(0);
  int st = 0;
  auto stage = [&](auto edge_stage) __attribute__((always_inline)) {
    wait_vmcnt<0>();  // this wave's part of the stage has landed
    stage_barrier();  // everyone's, and the stage before is used
    issue(st + 1);
    if (!busy) return;
    scores(edge_stage, st);
    values(edge_stage, st);
  };
  const int seen_whole = W.C / SP - W.first * (kGrain / SP);  // stages before the nodes
  const int inner = seen_whole < stages ? seen_whole : stages;
  for (; st < inner; ++st) stage(Bool<false>{});
  for (; st < stages; ++st) stage(Bool<true>{});
  wait_vmcnt<0>();  // the reads past the end have written their zeros
  __syncthreads();
  if (__any(any_odd != 0))
    add_odd<RT>(A, W, row0, n, o, [&](int e, int r) { return 16 * e + 4 * kg + r; },
                [&](int p) {
                  const int at = p / kGrain;
                  return at >= W.first && at < W.end && p / WP % PG == pg;
                });
  float* s_o = reinterpret_cast<float*>(s_buf);
  if (kg == 0)
#pragma unroll
    for (int t = 0; t < RT; ++t)
      s_m[wave * 16 * RT + 16 * t + n] = mx[t], s_l[wave * 16 * RT + 16 * t + n] = l[t][0];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (t) __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e)
      *reinterpret_cast<float4v*>(s_o + (wave * 16 + n) * kOPad + 16 * e + 4 * kg) = o[t][e];
    __syncthreads();
    finish<RG, PG>(A, W, s_o, s_m, s_l, t, 16 * RT);
  }
  __syncthreads();  // the next range's stages go where the rows are read from
  }
  share.rest(A, 32 * RG);
}

// The ranges' sums joined, of heads that several workgroups share: 32 threads per
// row, 4 elements each, G such groups taking every G-th range of it; a workgroup
// has 8 / G rows of one head.  Where there are few rows their ranges are many, and
// each costs the wait for a load.
template <int G>
__global__ __launch_bounds__(256) void join_kernel(Attend A, int per_head) {
  constexpr int kRows = 8 / G;
  __shared__ float4v s_x[G][kRows][32];
  __shared__ float s_m[G][kRows], s_s[G][kRows];
  const int bg = blockIdx.x / per_head, t = threadIdx.x >> 5, grp = t / kRows, rr = t - grp * kRows;
  const int row = kRows * (blockIdx.x - bg * per_head) + rr;
  const int b = bg / A.nkv, g = bg - b * A.nkv, n = grains_of(A, b);
  if (n == 0) return;
  const Split P(grains_below(A, A.B) * A.nkv, A.wgs);
  const int from = grains_below(A, b) * A.nkv + g * n;
  const int w0 = P.owner(from), k = P.owner(from + n - 1) - w0 + 1;
  if (k == 1) return;
  // the first range is its workgroup's second unless the head starts its share
  const long e0 = 2L * w0 + (P.from(w0) < from);
  const int d = 4 * (threadIdx.x & 31);
  const float* po = A.part + (long)(row < A.R ? row : 0) * kHd + d;
  const float* pm = A.part + 2 * (long)A.wgs * A.R * kHd + (long)(row < A.R ? row : 0) * 2;
  auto entry = [&](int i) { return (i == 0 ? e0 : 2L * (w0 + i)) * A.R; };
  float m = -__builtin_inff();
#pragma unroll 4
  for (int i = grp; i < k; i += G) m = fmaxf(m, pm[entry(i) * 2]);
  if (G > 1) {
    if (d == 0) s_m[grp][rr] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G; ++i) m = fmaxf(m, s_m[i][rr]);
  }
  const float ref = m == -__builtin_inff() ? 0.f : m;
  float sum = 0.f;
  float4v x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int i = grp; i < k; i += G) {
    const float al = __builtin_amdgcn_exp2f(pm[entry(i) * 2] - ref);
    sum += al * pm[entry(i) * 2 + 1];
    x += al * *reinterpret_cast<const float4v*>(po + entry(i) * kHd);
  }
  if (G > 1) {
    s_x[grp][rr][threadIdx.x & 31] = x;
    if (d == 0) s_s[grp][rr] = sum;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int i = 1; i < G; ++i) x += s_x[i][rr][threadIdx.x & 31], sum += s_s[i][rr];
  }
  if (row >= A.R) return;
  const int head = row / A.S, node = row - head * A.S;
  const u64* see = A.seen + ((A.trees > 1 ? (long)b * A.S : 0) + node) * kWords;
  const bool live = (see[node >> 6] >> (node & 63)) & 1;
  const float is = 1.f / sum;
  typedef h16 half4v __attribute__((ext_vector_type(4)));
  half4v y;
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = live ? (h16)(x[i] * is) : (h16)0.f;
  *reinterpret_cast<half4v*>(A.out + ((long)b * A.S + node) * A.ld_o +
                             (long)(g * A.rep + head) * kHd + d) = y;
}

// Rows per workgroup, and workgroups: as many as the chip holds at a time, two per
// CU (they share the work evenly), or one for each grain that there can be.  One
// per CU took 157 us for 8 sequences of 8000 with 64 nodes, two take 120.
// 64 or 128 rows, the other half of the waves on the other half of a stage or on
// rows of their own: of 32 sequences of 8000, 16 rows 222 / 258 us and 64 rows
// 239 / 252, and 68 rows, which take two workgroups of 64, 290 / 248.
struct Plan {
  int rows, blocks, wgs;
};
Plan plan_of(long B, long nkv, long rep, long S, long bound) {
  const long R = rep * S;
  Plan p;
  p.rows = R <= 64 ? 64 : 128;
  p.blocks = (int)((R + p.rows - 1) / p.rows);
  const long most = B * nkv * ((bound - 1) / kGrain + 1);
  const long fill = 2L * hn_device_cus() / p.blocks;
  p.wgs = (int)(most < fill ? most : fill < 1 ? 1 : fill);
  return p;
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

// See include/hn_int4.h.
extern "C" int hn_tree_plan(const int* parents, long ld_p, long B, long S, int* up, int* depth,
                            unsigned long long* seen, void* stream) {
  HN_ARG_CHECK(B >= 0 && S >= 1 && S <= kMaxNodes && ld_p >= S,
               "hn_tree_plan: need 1 <= nodes <= %d and ld_p >= nodes", kMaxNodes);
  if (B == 0) return 0;
  HN_ARG_CHECK(parents && up && depth && seen, "hn_tree_plan: null operand");
  hipLaunchKernelGGL(plan_kernel, dim3((unsigned)B), dim3(kMaxNodes), 0, (hipStream_t)stream,
                     parents, ld_p, (int)S, up, depth, seen);
  HN_LAUNCH_CHECK("hn_tree_plan");
  return 0;
}

// See include/hn_int4.h.
extern "C" int hn_tree_append(const void* qkv, long ld_qkv, const float* cos_t, const float* sin_t,
                              long table_rows, const int* depth, long trees, const long* lens,
                              long B, long S, long nkv, long rep, long hd, void* q_out, void* kt,
                              void* v, long max_len, void* stream) {
  const char* who = "hn_tree_append";
  HN_ARG_CHECK(B >= 0 && S >= 1 && S <= kMaxNodes && nkv > 0 && rep > 0 && hd == kHd,
               "%s: need head_dim %d, 1 <= nodes <= %d and nkv, rep > 0", who, kHd, kMaxNodes);
  HN_ARG_CHECK(trees == 1 || trees == B, "%s: need one tree or one per sequence", who);
  HN_ARG_CHECK(max_len > 0 && table_rows > 0 && ld_qkv >= (nkv * rep + 2 * nkv) * hd,
               "%s: qkv rows must hold q, k and v", who);
  if (B == 0) return 0;
  HN_ARG_CHECK(qkv && cos_t && sin_t && depth && lens && q_out && kt && v, "%s: null operand", who);
  HN_ARG_CHECK(B * S < (1L << 31) && nkv * (rep + 1) <= 65535, "%s: too many rows or heads", who);
  // Up to 40 nodes the launch's latency is all there is, and the kernel by elements
  // has less of it: 1, 32, 64, 256 and 512 nodes of 32 + 2 x 8 heads take it 2.0,
  // 2.9, 3.6, 8.0 and 16.1 us, the other 3.2, 3.1, 3.4, 3.7 and 4.4.  The crossing is
  // near 50 nodes there; with fewer heads it comes later, with more a little sooner,
  // and the rule is off by less than a microsecond: 64 and 256 nodes of 1 + 2 heads
  // 2.4 and 2.5 us by elements, 3.0 and 3.1 by rows; of 8 + 2 x 2 heads 2.4 and 3.6, 3.3
  // and 3.4; 32 nodes of 96 + 2 x 8 heads 3.8 by elements, where 64 take 3.5 by rows.
  if (B * S > 40 && ld_qkv % 8 == 0 && al16(qkv) && al16(cos_t) && al16(sin_t) && al16(q_out) && al16(v)) {
    hipLaunchKernelGGL(append_rows_kernel,
                       dim3((unsigned)((B * S + kAppend - 1) / kAppend),
                            (unsigned)((nkv * rep + kHeads - 1) / kHeads + nkv)),
                       dim3(256), 0, (hipStream_t)stream, (const h16*)qkv, ld_qkv, cos_t, sin_t,
                       table_rows, depth, (int)trees, lens, (int)B, (int)S, (int)nkv, (int)rep,
                       (h16*)q_out, (h16*)kt, (h16*)v, max_len);
    HN_LAUNCH_CHECK(who);
    return 0;
  }
  hipLaunchKernelGGL(append_kernel, dim3((unsigned)(B * S), (unsigned)(nkv * (rep + 1))), dim3(kHd),
                     0, (hipStream_t)stream, (const h16*)qkv, ld_qkv, cos_t, sin_t, table_rows, depth,
                     (int)trees, lens, (int)S, (int)nkv, (int)rep, (h16*)q_out, (h16*)kt, (h16*)v,
                     max_len);
  HN_LAUNCH_CHECK(who);
  return 0;
}

// See include/hn_int4.h.
extern "C" long hn_tree_attention_workspace_bytes(long B, long nkv, long rep, long S, long bound) {
  if (B <= 0 || nkv <= 0 || rep <= 0 || S <= 0 || bound <= 0) return 0;
  const Plan p = plan_of(B, nkv, rep, S, bound);
  return bound <= kGrain ? 0 : 2L * p.wgs * rep * S * (kHd + 2) * 4;
}

// See include/hn_int4.h.
extern "C" int hn_tree_attention(const void* q, const void* kt, const void* v, long max_len,
                                 const long* lens, const unsigned long long* seen, long trees,
                                 long B, long nkv, long rep, long hd, long S, long bound,
                                 float scale, void* out, long ld_o, void* work, long work_bytes,
                                 void* stream) {
  const char* who = "hn_tree_attention";
  HN_ARG_CHECK(B >= 0 && S >= 1 && S <= kMaxNodes && nkv > 0 && rep > 0 && hd == kHd,
               "%s: need head_dim %d, 1 <= nodes <= %d and nkv, rep > 0", who, kHd, kMaxNodes);
  HN_ARG_CHECK(trees == 1 || trees == B, "%s: need one tree or one per sequence", who);
  HN_ARG_CHECK(bound >= S && bound <= max_len && max_len % 8 == 0 && max_len < (1L << 23),
               "%s: need nodes <= bound <= max_len, max_len %% 8 == 0, below 2^23", who);
  if (B == 0) return 0;
  HN_ARG_CHECK(q && kt && v && lens && seen && out, "%s: null operand", who);
  // (the kernel masks scores and takes their maximum before it scales them)
  HN_ARG_CHECK(scale > 0.f && scale <= FLT_MAX / kLog2e, "%s: scale must be finite and above 0",
               who);
  HN_ARG_CHECK(al16(q) && al16(kt) && al16(v) && al16(out) && ld_o % 8 == 0 &&
                   ld_o >= nkv * rep * hd,
               "%s: operands must be 16-byte aligned, ld_o >= heads * %d", who, kHd);
  const Plan p = plan_of(B, nkv, rep, S, bound);
  const long R = rep * S;
  HN_ARG_CHECK(B * nkv * ((bound + kGrain - 1) / kGrain) < (1L << 31) &&
                   B * nkv * R < (1L << 31) && (p.wgs + 7L) / 8 * 8 * p.blocks < (1L << 31),
               "%s: too many rows", who);
  const long need = hn_tree_attention_workspace_bytes(B, nkv, rep, S, bound);
  HN_ARG_CHECK(need == 0 || (work && al16(work) && work_bytes >= need),
               "%s: needs a 16-byte aligned workspace of %ld bytes (got %ld)", who, need,
               work_bytes);
  const Attend A = {(const h16*)q, (const h16*)kt, (const h16*)v, lens, seen, (h16*)out,
                    (float*)work, max_len, bound, ld_o, (int)trees, (int)B, (int)nkv, (int)rep,
                    (int)S, (int)R, p.blocks, p.wgs, scale};
  const dim3 grid((unsigned)((p.wgs + 7) / 8 * 8 * p.blocks));
  hipStream_t st = (hipStream_t)stream;
  const auto kern = p.rows == 64 ? share_kernel<2, 2> : share_kernel<4, 1>;
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, A);
  HN_LAUNCH_CHECK(who);
  if (need) {  // a head of several grains may be shared
    // whole calls: 512 rows 15.1 / 14.4 us (G = 1 / 8) over 1500 positions, 1024 rows
    // 63 / 52 over 30000, 2048 rows of 8 sequences 24 / 26, 8192 rows 37 / 44
    const bool few = B * nkv * R <= 1024;
    const auto join = few ? join_kernel<8> : join_kernel<1>;
    const long per_head = few ? R : (R + 7) / 8;
    hipLaunchKernelGGL(join, dim3((unsigned)(B * nkv * per_head)), dim3(256), 0, st, A,
                       (int)per_head);
    HN_LAUNCH_CHECK(who);
  }
  return 0;
}
