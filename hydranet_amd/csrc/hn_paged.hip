// A paged KV cache: the append of a step's keys and values with the position
// rotation of its queries and keys, and the attention over the pages.
//
// A page holds `page` positions of every KV head: keys [page id][kv head][slot][hd],
// values [page id][kv head][slot / 8][hd][8].  Row b of the table names the pages of
// sequence b in order.  A sequence with C = lens[b] >= 0 cached positions adds rows
// starts[b] to starts[b + 1] of the step (one row, b, without starts) at positions C on;
// a row sees the positions up to its own.
#include "hn_paged.h"

namespace {

// One thread per element, grid (T, nh + 2 nkv).
template <class T>
__global__ __launch_bounds__(256) void append_kernel(Step P, const T* __restrict__ qkv, long ld,
                                                     const float* __restrict__ cos_t,
                                                     const float* __restrict__ sin_t, long rows,
                                                     int rd, int pairs, int nh, int hd,
                                                     T* __restrict__ q_out, T* __restrict__ k,
                                                     T* __restrict__ v) {
  const int t = blockIdx.x, head = blockIdx.y, d = threadIdx.x;
  const Row r = row_of(P, t);
  if (r.b < 0 || d >= hd) return;
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

// One wave per (row, query head).
template <class T, int HD>
__global__ __launch_bounds__(64) void attend_kernel(Step P, const T* __restrict__ q, long ld_q,
                                                    const T* __restrict__ k,
                                                    const T* __restrict__ v, int rep, float scale,
                                                    T* __restrict__ out, long ld_o) {
  __shared__ float s_q[HD], s_p[64];
  __shared__ long s_pg[64];
  const int t = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, g = head / rep;
  const Row r = row_of(P, t);
  if (r.b < 0) return;
  for (int d = lane; d < HD; d += 64) s_q[d] = (float)q[(long)t * ld_q + (long)head * HD + d];
  float m = -__builtin_inff(), sum = 0.f, o[HD / 64] = {};
  // the sequence's positions with its last row: all on pages that are named, or none is read
  const long L = r.pos < 0 ? 0 : r.pos + (P.starts ? min(P.starts[r.b + 1], P.T) - t : 1);
  bool bad = L > P.cols * P.page;
  for (long p0 = lane * (long)P.page; !bad && p0 < L; p0 += 64 * P.page)
    bad = page_of(P, r.b, p0) < 0;
  bad = __any(bad);
  for (long p0 = 0; !bad && p0 <= r.pos; p0 += 64) {
    const long p = p0 + lane;
    float s = -__builtin_inff();
    long pg = 0;
    if (p <= r.pos) {
      pg = page_of(P, r.b, p);
      const T* kp = k + ((pg * P.nkv + g) * P.page + (p & (P.page - 1))) * HD;
      s = 0.f;
      for (int d = 0; d < HD; ++d) s += s_q[d] * (float)kp[d];
      s *= scale;
    }
    float top = s;
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float nm = fmaxf(m, top), al = __expf(m - nm);
    const float e = p <= r.pos ? __expf(s - nm) : 0.f;
    m = nm;
    __syncthreads();
    s_p[lane] = e, s_pg[lane] = pg;
    __syncthreads();
    sum *= al;
    for (int i = 0; i < HD / 64; ++i) o[i] *= al;
    for (int j = 0; j < 64 && p0 + j <= r.pos; ++j) {
      const int slot = (int)((p0 + j) & (P.page - 1));
      const T* vp = v + ((s_pg[j] * P.nkv + g) * P.page + (slot & ~7)) * HD + (slot & 7);
      sum += s_p[j];
      for (int i = 0; i < HD / 64; ++i) o[i] += s_p[j] * (float)vp[(lane + 64 * i) * 8];
    }
  }
  for (int i = 0; i < HD / 64; ++i)
    out[(long)t * ld_o + (long)head * HD + lane + 64 * i] =
        (T)(r.pos < 0 ? 0.f : bad ? __builtin_nanf("") : o[i] / sum);
}

// Pages src[i] to dst[i] of every layer; the addresses and pairs go in the arguments.
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

int check_step(const char* who, const Step& P, const void* qkv, const void* k, const void* v,
               long nh, long hd, long T, int dtype) {
  HN_ARG_CHECK(dtype == 0 || dtype == 1, "%s: dtype %d (0 fp16, 1 bf16)", who, dtype);
  HN_ARG_CHECK(P.nkv > 0 && nh > 0 && nh % P.nkv == 0 && nh < 1 << 16,
               "%s: %ld heads over %d KV heads", who, nh, P.nkv);
  HN_ARG_CHECK(fits(hd, P.page), "%s: heads of 64, 128 or 256 (got %ld), pages of 16 to 1024 "
               "positions, a power of two (got %d)", who, hd, P.page);
  HN_ARG_CHECK(P.B >= 0 && T >= 0 && T < 1 << 30 && P.pages >= 0 && P.cols >= 0 &&
                   P.ld >= P.cols && (P.starts || T == P.B),
               "%s: %d sequences, %ld rows, %ld pages, a table of %ld columns (row %ld)", who, P.B,
               T, P.pages, P.cols, P.ld);
  if (P.B == 0 || T == 0) return 0;
  HN_ARG_CHECK(qkv && k && v && P.table && P.lens, "%s: null operand", who);
  HN_ARG_CHECK((uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0, "%s: pages not 16-byte aligned",
               who);
  return 0;
}

Step step_of(const int* table, long ld_table, long cols, long num_pages, const long* lens,
             const int* starts, long B, long T, long nkv, long page) {
  return Step{table, ld_table, cols, num_pages, lens, starts, (int)B, (int)T, (int)nkv, (int)page};
}

template <class T>
int append(const Step& P, const void* qkv, long ld, const float* cos_t, const float* sin_t,
           long rows, int rd, int pairs, int nh, int hd, void* q_out, void* k, void* v,
           hipStream_t stream) {
  append_kernel<T><<<dim3(P.T, nh + 2 * P.nkv), hd, 0, stream>>>(
      P, (const T*)qkv, ld, cos_t, sin_t, rows, rd, pairs, nh, hd, (T*)q_out, (T*)k, (T*)v);
  HN_LAUNCH_CHECK("hn_paged_append");
  return 0;
}

template <class T>
int attend(const Step& P, const void* q, long ld_q, const void* k, const void* v, int nh, int hd,
           float scale, void* out, long ld_o, hipStream_t stream) {
  const dim3 grid(P.T, nh);
  const int rep = nh / P.nkv;
#define HN_ATTEND(HD)                                                                     \
  attend_kernel<T, HD><<<grid, 64, 0, stream>>>(P, (const T*)q, ld_q, (const T*)k,        \
                                                (const T*)v, rep, scale, (T*)out, ld_o)
  if (hd == 64) HN_ATTEND(64);
  else if (hd == 128) HN_ATTEND(128);
  else HN_ATTEND(256);
#undef HN_ATTEND
  HN_LAUNCH_CHECK("hn_paged_attention");
  return 0;
}

}  // namespace

extern "C" int hn_paged_append(const void* qkv, long ld_qkv, int dtype, const float* cos_t,
                               const float* sin_t, long table_rows, long rotary, int interleaved,
                               const int* table, long ld_table, long cols, long num_pages,
                               const long* lens, const int* starts, long B, long T, long nh,
                               long nkv, long hd, long page, void* q_out, void* k, void* v,
                               void* stream) {
  const Step P = step_of(table, ld_table, cols, num_pages, lens, starts, B, T, nkv, page);
  if (int rc = check_step("hn_paged_append", P, qkv, k, v, nh, hd, T, dtype)) return rc;
  HN_ARG_CHECK(rotary >= 0 && rotary <= hd && rotary % 2 == 0 && table_rows >= 0,
               "hn_paged_append: %ld rotated dimensions of %ld, %ld positions", rotary, hd,
               table_rows);
  if (B == 0 || T == 0) return 0;
  HN_ARG_CHECK(q_out && (rotary == 0 || (cos_t && sin_t)), "hn_paged_append: null operand");
  HN_ARG_CHECK(ld_qkv >= (nh + 2 * nkv) * hd, "hn_paged_append: rows of %ld, a stride of %ld",
               (nh + 2 * nkv) * hd, ld_qkv);
  return (dtype == 0 ? append<h16> : append<b16>)(P, qkv, ld_qkv, cos_t, sin_t, table_rows,
                                                  (int)rotary, interleaved, (int)nh, (int)hd,
                                                  q_out, k, v, (hipStream_t)stream);
}

extern "C" long hn_paged_attention_workspace_bytes(long B, long T, long nh, long nkv, long hd,
                                                   long max_new, long bound) {
  return 0;
}

extern "C" int hn_paged_attention(const void* q, long ld_q, int dtype, const void* k,
                                  const void* v, const int* table, long ld_table, long cols,
                                  long num_pages, const long* lens, const int* starts, long B,
                                  long T, long nh, long nkv, long hd, long page, long max_new,
                                  long bound, float scale, void* out, long ld_o, void* work,
                                  long work_bytes, void* stream) {
  const Step P = step_of(table, ld_table, cols, num_pages, lens, starts, B, T, nkv, page);
  if (int rc = check_step("hn_paged_attention", P, q, k, v, nh, hd, T, dtype)) return rc;
  HN_ARG_CHECK(max_new >= 1 && bound >= 1, "hn_paged_attention: max_new %ld, bound %ld", max_new,
               bound);
  HN_ARG_CHECK(scale > 0.f && scale * 1.4426950408889634f < __builtin_inff(),
               "hn_paged_attention: scale %g", (double)scale);
  if (B == 0 || T == 0) return 0;
  HN_ARG_CHECK(out && ld_q >= nh * hd && ld_o >= nh * hd && ld_q % 8 == 0 && ld_o % 8 == 0 &&
                   (uintptr_t)q % 16 == 0 && (uintptr_t)out % 16 == 0,
               "hn_paged_attention: rows of %ld, strides of %ld and %ld: 16-byte aligned rows",
               nh * hd, ld_q, ld_o);
  return (dtype == 0 ? attend<h16> : attend<b16>)(P, q, ld_q, k, v, (int)nh, (int)hd, scale, out,
                                                  ld_o, (hipStream_t)stream);
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
