// Attention of a tree of drafted tokens over the KV cache: the plan of a tree,
// RoPE and the cache append of its nodes, and the attention.
//
// A tree is a row of parents, node i below parents[i] < i (-1: directly below
// the cached positions).  A node with any other parent, and every node below
// it, is padding.  Node i of a sequence with C = lens[b] cached positions sits
// at cache position C + i, its rotary position is C + depth(i), and it sees
// positions [0, C) and those of itself and its ancestors.
#include "hn_common.h"

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

// Grid (B * S, nh + nkv), a thread per element of a head.
__global__ __launch_bounds__(kHd) void append_kernel(
    const h16* __restrict__ qkv, long ld, const float* __restrict__ cos_t,
    const float* __restrict__ sin_t, long table_rows, const int* __restrict__ depth, int trees,
    const long* __restrict__ lens, int S, int nkv, int rep, h16* __restrict__ q_out,
    h16* __restrict__ kt, h16* __restrict__ vc, long max_len) {
  const int row = blockIdx.x, head = blockIdx.y, d = threadIdx.x;
  const int b = row / S, i = row - b * S, nh = nkv * rep;
  const int dep = depth[(trees > 1 ? (long)b * S : 0) + i];
  const long C = lens[b], pos = C + dep, slot = C + i;
  const bool live = C >= 0 && dep >= 0;
  const bool in = live && pos < table_rows && slot < max_len;
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

// One wave per (sequence, query head, node): 64 positions at a time, a lane per
// position for the scores, then a lane per two elements of the output.
__global__ __launch_bounds__(256) void attend_kernel(
    const h16* __restrict__ q, const h16* __restrict__ ktc, const h16* __restrict__ vc,
    long max_len, const long* __restrict__ lens, const u64* __restrict__ seen, int trees, long rows,
    int nkv, int rep, int S, long bound, float scale, h16* __restrict__ out, long ld_o) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);  // (b, g, r, i)
  if (row >= rows) return;
  const int i = (int)(row % S);
  const long bh = row / S, bg = bh / rep, b = bg / nkv;
  const int head = (int)(bh - b * nkv * rep);
  const u64* see = seen + ((trees > 1 ? b * S : 0) + i) * kWords;
  const long C = lens[b], L = C + S;
  h16* o = out + (b * S + i) * ld_o + (long)head * kHd + 2 * lane;
  const bool live = C >= 0 && ((see[i >> 6] >> (i & 63)) & 1);
  if (!live || L > bound) {
    const h16 v = live ? (h16)__builtin_nanf("") : (h16)0.f;
    o[0] = v, o[1] = v;
    return;
  }
  const h16* kt = ktc + bg * kHd * max_len;
  const h16* v = vc + bg * max_len * kHd;
  const h16* qr = q + row * kHd;
  float mx = -__builtin_inff(), sum = 0.f, o0 = 0.f, o1 = 0.f;
  for (long p0 = 0; p0 < L; p0 += 64) {
    const long p = p0 + lane;
    bool vis = p < C;
    if (p >= C && p < L) vis = (see[(p - C) >> 6] >> ((p - C) & 63)) & 1;
    float s = -__builtin_inff();
    if (vis) {
      s = 0.f;
      for (int d = 0; d < kHd; ++d) s += (float)qr[d] * (float)kt[(long)d * max_len + p];
      s *= scale;
    }
    float tm = s;
    for (int off = 32; off; off >>= 1) tm = fmaxf(tm, __shfl_xor(tm, off, 64));
    const float nm = fmaxf(mx, tm), ref = nm == -__builtin_inff() ? 0.f : nm;
    const float al = expf(mx - ref), e = vis ? expf(s - ref) : 0.f;
    sum = sum * al + e, o0 *= al, o1 *= al, mx = nm;
    u64 todo = __ballot(vis);
    while (todo) {
      const int j = __builtin_ctzll(todo);
      todo &= todo - 1;
      const float pj = __shfl(e, j, 64);
      const h16* vr = v + (p0 + j) * kHd + 2 * lane;
      o0 += pj * (float)vr[0], o1 += pj * (float)vr[1];
    }
  }
  for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off, 64);
  o[0] = (h16)(o0 / sum), o[1] = (h16)(o1 / sum);
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
  hipLaunchKernelGGL(append_kernel, dim3((unsigned)(B * S), (unsigned)(nkv * (rep + 1))), dim3(kHd),
                     0, (hipStream_t)stream, (const h16*)qkv, ld_qkv, cos_t, sin_t, table_rows, depth,
                     (int)trees, lens, (int)S, (int)nkv, (int)rep, (h16*)q_out, (h16*)kt, (h16*)v,
                     max_len);
  HN_LAUNCH_CHECK(who);
  return 0;
}

// See include/hn_int4.h.
extern "C" long hn_tree_attention_workspace_bytes(long B, long nkv, long rep, long S, long bound) {
  return 0;
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
  HN_ARG_CHECK(al16(q) && al16(kt) && al16(v) && al16(out) && ld_o % 8 == 0 &&
                   ld_o >= nkv * rep * hd && lens && seen,
               "%s: operands must be 16-byte aligned, ld_o >= heads * %d", who, kHd);
  const long rows = B * nkv * rep * S;
  HN_ARG_CHECK(rows < (1L << 31), "%s: too many rows", who);
  hipLaunchKernelGGL(attend_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0,
                     (hipStream_t)stream, (const h16*)q, (const h16*)kt, (const h16*)v, max_len, lens,
                     seen, (int)trees, rows, (int)nkv, (int)rep, (int)S, bound, scale, (h16*)out,
                     ld_o);
  HN_LAUNCH_CHECK(who);
  return 0;
}
