// The KV cache's positions compacted after drafted tokens were verified, and
// copied to further sequences, in every layer by one launch (up to 64 layers,
// whose addresses travel in the kernel's arguments).  Keys are cached
// [B][nkv][hd][max_len], values [B][nkv][max_len][hd], fp16.
#include "hn_common.h"

namespace {

constexpr int kLayers = 64;  // layers per launch
constexpr int kPairs = 128;  // copies per launch

struct Layers {
  h16* kt[kLayers];
  h16* v[kLayers];
};

// Grid (B * nkv, layers, 2): keys, values.  Positions go in ascending order, kStep at
// a time: the sources of a step are read before its destinations are written, and
// path[j] >= j, so a later source (at or past its own j) is never an earlier
// destination.  Of the keys, which lie 2 bytes to a row, 8 lanes take a row's step,
// whose destinations are next to each other: a thread per row, 8 moves in flight,
// asked the caches for 8 times the lines (94 us for the 74 below).
// Bound by memory's requests, not its bytes: a position's 128 elements lie in as many
// rows of K^T, 2 bytes of each.  32 sequences, 32 layers of 8 heads, 128 moved
// positions: 73 us, in which 88 MB are fetched and 53 MB written for 34 MB of moves,
// 29 us at a copy's rate.  Of the 1.13 million writes that reach memory 0.97 million
// are parts of a 64-byte line, and the waves wait during 84 % of their cycles.  Threads that read and wrote
// whole lines of a row, 64 or 128 bytes, took 139 and 266 us; 256 threads for 128
// rows 77, 8 rows in flight per lane 73, two layers per workgroup 66 (but the same as
// before on a cache that was not just read, 87 us a call).
constexpr int kStep = 8;
__global__ __launch_bounds__(256) void keep_kernel(Layers L, long max_len, int nkv, int hd,
                                                   const long* __restrict__ lens,
                                                   const int* __restrict__ path, long ld_p,
                                                   const int* __restrict__ count, int S,
                                                   long* __restrict__ lens_out) {
  constexpr int kRows = 4;  // rows of keys in flight per lane
  const int bg = blockIdx.x, b = bg / nkv, layer = blockIdx.y, tid = threadIdx.x;
  const long C = lens[b];
  int n = count[b];
  n = n < 0 ? 0 : n > S ? S : n;
  if (lens_out && layer == 0 && bg == b * nkv && blockIdx.z == 0 && tid == 0)
    lens_out[b] = C < 0 ? C : C + n;
  if (C < 0) return;
  const long left = max_len - C;
  const int* p = path + (long)b * ld_p;
  if (blockIdx.z == 0) {
    h16* kt = L.kt[layer] + (long)bg * hd * max_len + C;
    const int j = tid & (kStep - 1), r = tid / kStep, rows = blockDim.x / kStep;
    for (int j0 = 0; j0 < n; j0 += kStep) {
      const int to = j0 + j, at = to < n ? p[to] : 0;
      const bool moves = at > to && at < left;
      for (int d0 = r; d0 < hd; d0 += kRows * rows) {
        h16 x[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (moves && d0 + i * rows < hd) x[i] = kt[(long)(d0 + i * rows) * max_len + at];
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (moves && d0 + i * rows < hd) kt[(long)(d0 + i * rows) * max_len + to] = x[i];
      }
    }
    return;
  }
  h16* v = L.v[layer] + ((long)bg * max_len + C) * hd;
  for (int d = tid; d < hd; d += blockDim.x)
    for (int j0 = 0; j0 < n; j0 += kStep) {
      h16 x[kStep];
      int at[kStep];
#pragma unroll
      for (int j = 0; j < kStep; ++j) {
        at[j] = j0 + j < n ? p[j0 + j] : 0;
        if (at[j] > j0 + j && at[j] < left) x[j] = v[(long)at[j] * hd + d];
      }
#pragma unroll
      for (int j = 0; j < kStep; ++j)
        if (at[j] > j0 + j && at[j] < left) v[(long)(j0 + j) * hd + d] = x[j];
    }
}

// Copies, those of one source next to each other: sources src[g], destinations
// dst[first[g] .. first[g + 1]).
struct Copies {
  int src[kPairs], first[kPairs + 1], dst[kPairs];
};

// By elements, for layers of any alignment: grid (nkv * hd, sources, layers), the
// positions of one row of keys and as many elements of the values.
__global__ __launch_bounds__(256) void fork_kernel(Layers L, Copies P, long max_len, int nkv, int hd,
                                                   long n) {
  const int g = blockIdx.x / hd, d = blockIdx.x - g * hd, layer = blockIdx.z;
  const long a = (long)P.src[blockIdx.y] * nkv + g;
  h16* kt = L.kt[layer];
  h16* v = L.v[layer];
  for (long p = threadIdx.x; p < n; p += blockDim.x) {
    const h16 kx = kt[(a * hd + d) * max_len + p], vx = v[a * max_len * hd + d * n + p];
    for (int i = P.first[blockIdx.y]; i < P.first[blockIdx.y + 1]; ++i) {
      const long b = (long)P.dst[i] * nkv + g;
      kt[(b * hd + d) * max_len + p] = kx;
      v[b * max_len * hd + d * n + p] = vx;
    }
  }
}

// By vectors of 16 bytes, one per thread, stored to every destination past the
// caches (non-temporal: what is written is many times what they hold).  Grid
// (workgroups of keys, then of values; sources; layers).  The last vector of a row
// of keys may hold positions past n, which stay as they are in the destination.
// Bound by HBM: 2 prompts of 1901 positions to 5 sequences each, 32 layers of 8
// heads, 588 us for 3.0 GB (5.1 TB/s, a large copy's 4.9).  Whole calls, timed on
// one day: 603 us; with 8, 4, 2 vectors per thread and plain stores 673, 635, 622,
// with 2 and 4 non-temporal 615, 624.
__global__ __launch_bounds__(256) void fork_vec_kernel(Layers L, Copies P, long max_len, int nkv,
                                                       int hd, int n, int key_groups) {
  const int layer = blockIdx.z, sg = blockIdx.y;
  const bool keys = (int)blockIdx.x < key_groups;
  const int nv = keys ? (n + 7) / 8 : n * (hd / 8);  // vectors of a row
  const long idx = (long)(blockIdx.x - (keys ? 0 : key_groups)) * 256 + threadIdx.x;
  const long row = idx / nv, col = idx - row * nv;
  if (row >= (keys ? nkv * hd : nkv)) return;
  h16* base = keys ? L.kt[layer] : L.v[layer];
  const long seq = (long)nkv * hd * max_len, at = row * (keys ? max_len : max_len * hd) + 8 * col;
  const u32x4 x = *reinterpret_cast<const u32x4*>(base + P.src[sg] * seq + at);
  const int tail = keys && col == nv - 1 && n % 8 ? n % 8 : 8;
  for (int k = P.first[sg]; k < P.first[sg + 1]; ++k) {
    h16* out = base + P.dst[k] * seq + at;
    if (tail == 8) {
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(out));
    } else {
      const half8_t h = __builtin_bit_cast(half8_t, x);
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < tail) out[e] = h[e];
    }
  }
}

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

// See include/hn_int4.h.
extern "C" int hn_kv_keep(void* const* kt, void* const* v, long layers, long max_len, long B,
                          long nkv, long hd, const long* lens, const int* path, long ld_path,
                          const int* count, long S, long* lens_out, void* stream) {
  const char* who = "hn_kv_keep";
  HN_ARG_CHECK(layers >= 1 && B >= 0 && nkv > 0 && hd > 0 && max_len > 0 && S >= 1 && ld_path >= S,
               "%s: need layers, heads, positions and nodes > 0, ld_path >= nodes", who);
  HN_ARG_CHECK(B * nkv < (1L << 31), "%s: too many heads", who);
  if (B == 0) return 0;
  HN_ARG_CHECK(kt && v && lens && path && count, "%s: null operand", who);
  HN_ARG_CHECK(lens_out != lens, "%s: lens_out must not be lens (other workgroups read it)", who);
  for (long l = 0; l < layers; ++l) HN_ARG_CHECK(kt[l] && v[l], "%s: null layer %ld", who, l);
  for (long l0 = 0; l0 < layers; l0 += kLayers) {
    const int m = (int)(layers - l0 < kLayers ? layers - l0 : kLayers);
    Layers L = {};
    for (int l = 0; l < m; ++l) L.kt[l] = (h16*)kt[l0 + l], L.v[l] = (h16*)v[l0 + l];
    hipLaunchKernelGGL(keep_kernel, dim3((unsigned)(B * nkv), (unsigned)m, 2),
                       dim3(hd <= 128 ? 128 : 256), 0, (hipStream_t)stream, L, max_len, (int)nkv,
                       (int)hd, lens, path, ld_path, count, (int)S, l0 ? nullptr : lens_out);
    HN_LAUNCH_CHECK(who);
  }
  return 0;
}

// See include/hn_int4.h.
extern "C" int hn_kv_fork(void* const* kt, void* const* v, long layers, long max_len, long B,
                          long nkv, long hd, const int* src, const int* dst, long pairs, long n,
                          void* stream) {
  const char* who = "hn_kv_fork";
  HN_ARG_CHECK(layers >= 1 && B >= 0 && nkv > 0 && hd > 0 && max_len > 0 && pairs >= 0,
               "%s: need layers, heads and positions > 0", who);
  HN_ARG_CHECK(n >= 0 && n <= max_len, "%s: need 0 <= positions <= max_len", who);
  if (pairs == 0 || n == 0) return 0;
  HN_ARG_CHECK(nkv * hd < (1L << 31), "%s: too many heads", who);
  HN_ARG_CHECK(kt && v && src && dst, "%s: null operand", who);
  for (long l = 0; l < layers; ++l) HN_ARG_CHECK(kt[l] && v[l], "%s: null layer %ld", who, l);
  for (long i = 0; i < pairs; ++i) {
    HN_ARG_CHECK(src[i] >= 0 && src[i] < B && dst[i] >= 0 && dst[i] < B,
                 "%s: sequence out of range", who);
    for (long j = 0; j < pairs; ++j)
      HN_ARG_CHECK(dst[i] != src[j] && (i == j || dst[i] != dst[j]),
                   "%s: a destination is a source or given twice", who);
  }
  bool vec = max_len % 8 == 0 && hd % 8 == 0 && nkv * hd * n < (1L << 34);
  for (long l = 0; l < layers; ++l) vec = vec && al16(kt[l]) && al16(v[l]);
  for (long p0 = 0; p0 < pairs; p0 += kPairs) {
    const int np = (int)(pairs - p0 < kPairs ? pairs - p0 : kPairs);
    Copies P = {};
    int ns = 0, nd = 0;
    bool done[kPairs] = {};
    for (int p = 0; p < np; ++p) {
      if (done[p]) continue;
      P.src[ns] = src[p0 + p], P.first[ns] = nd;
      for (int r = p; r < np; ++r)
        if (!done[r] && src[p0 + r] == src[p0 + p]) P.dst[nd++] = dst[p0 + r], done[r] = true;
      P.first[++ns] = nd;
    }
    for (long l0 = 0; l0 < layers; l0 += kLayers) {
      const int m = (int)(layers - l0 < kLayers ? layers - l0 : kLayers);
      Layers L = {};
      for (int l = 0; l < m; ++l) L.kt[l] = (h16*)kt[l0 + l], L.v[l] = (h16*)v[l0 + l];
      if (vec) {
        const long kc = (nkv * hd * ((n + 7) / 8) + 255) / 256,
                   vc = (nkv * n * (hd / 8) + 255) / 256;
        hipLaunchKernelGGL(fork_vec_kernel, dim3((unsigned)(kc + vc), (unsigned)ns, (unsigned)m),
                           dim3(256), 0, (hipStream_t)stream, L, P, max_len, (int)nkv, (int)hd,
                           (int)n, (int)kc);
      } else {
        hipLaunchKernelGGL(fork_kernel, dim3((unsigned)(nkv * hd), (unsigned)ns, (unsigned)m),
                           dim3(256), 0, (hipStream_t)stream, L, P, max_len, (int)nkv, (int)hd, n);
      }
      HN_LAUNCH_CHECK(who);
    }
  }
  return 0;
}
