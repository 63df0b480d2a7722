// Logits adjusted before a token is drawn from them: penalties for tokens that the
// text holds, biases, and the tokens that a grammar allows.  One pass over the logits;
// what the text holds is counted on the way, so that no table of counts is kept.  Bound by
// the logits' bytes where they are many (64 rows of 130001 in fp32, texts to 4000, biases
// and bits: 20 to 21.5 us, 3.2 to 3.4 TB/s, a large copy moves 5.1), else by a launch and the
// latency of the text behind its length (64 rows of 32000, texts to 8000: 9.4 us; one row of
// 32000 3 us).
#include "hn_paged.h"

namespace {

struct Adjust {
  const long* text;  // [B][ld_text], width columns
  long ld_text, width;
  const long *lens, *first;
  const float *rep, *pres, *freq;  // [B] or null: the numbers
  float rep1, pres1, freq1;
  const long* ids;  // [B][ld_bias], n of them
  const float* bias;
  long ld_ids, ld_bias, n;
  const int* allowed;
  long ld_allowed;
  long V;
};

constexpr int kThreads = 1024;
constexpr uint32_t kSeen = 1u << 31;

// N elements at any alignment of the element's own.
template <class T, int N>
struct Some {
  T x[N];
};
template <class T, int N>
__device__ __forceinline__ Some<T, N> read(const T* p) {
  Some<T, N> s;
  __builtin_memcpy(&s, p, sizeof s);
  return s;
}

// A workgroup takes kThreads * N tokens of a row, N neighbours a thread.  How often each
// is in the text is gathered in LDS from the whole text (integers, so any order gives the
// same), and of several biases for a token the last one's index.  The logits are on their
// way meanwhile.
template <class T, int N>
__global__ __launch_bounds__(kThreads) void adjust_kernel(Adjust A, const T* logits, long ld,
                                                          T* out, long ld_o) {
  extern __shared__ __align__(16) uint32_t s_count[];
  typedef uint32_t Words __attribute__((ext_vector_type(N)));
  constexpr int kChunk = kThreads * N;
  int* s_bias = reinterpret_cast<int*>(s_count + kChunk);
  const int b = blockIdx.y, tid = threadIdx.x;
  const long v0 = (long)blockIdx.x * kChunk, v = v0 + tid * N;
  const T* src = logits + b * ld + v;
  T x[N];
  const bool whole = v + N <= A.V;
  if (whole) {
    const Some<T, N> s = read<T, N>(src);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = s.x[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = v + i < A.V ? src[i] : (T)0.f;
  }
  // (N neighbours' bits lie in one word: v is a multiple of N)
  const uint32_t word = A.allowed && v < A.V ? A.allowed[b * A.ld_allowed + (v >> 5)] : ~0u;
  const float r = A.rep ? A.rep[b] : A.rep1, pres = A.pres ? A.pres[b] : A.pres1;
  const float freq = A.freq ? A.freq[b] : A.freq1;
  const bool counts = A.text != nullptr, biases = A.n > 0;
  if (counts || biases) {
    *reinterpret_cast<Words*>(s_count + tid * N) = Words{};
    if (biases) *reinterpret_cast<Words*>(s_bias + tid * N) = Words{} - 1;
    __syncthreads();
    if (counts) {
      long n = A.lens ? A.lens[b] : A.width;
      n = n < A.width ? n : A.width;
      const long first = A.first ? A.first[b] : 0;
      const long* text = A.text + b * A.ld_text;
      auto count = [&](long token, long i) {
        const unsigned long at = (unsigned long)(token - v0);
        if (at >= kChunk) return;
        if (i < first) atomicOr(&s_count[at], kSeen);
        else atomicAdd(&s_count[at], 1u);
      };
      long i = 2 * tid;
      for (; i + 6 * kThreads + 1 < n; i += 8 * kThreads) {
        Some<long, 2> t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = read<long, 2>(text + i + 2 * j * kThreads);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          count(t[j].x[0], i + 2 * j * kThreads);
          count(t[j].x[1], i + 2 * j * kThreads + 1);
        }
      }
      for (; i < n; i += 2 * kThreads) {
        count(text[i], i);
        if (i + 1 < n) count(text[i + 1], i + 1);
      }
    }
    for (long i = tid; i < A.n; i += kThreads) {
      const unsigned long at = (unsigned long)(A.ids[b * A.ld_ids + i] - v0);
      if (at < kChunk) atomicMax(&s_bias[at], (int)i);
    }
    __syncthreads();
  }
  Words many = Words{}, last = Words{} - 1;
  if (counts) many = *reinterpret_cast<const Words*>(s_count + tid * N);
  if (biases) last = *reinterpret_cast<const Words*>(s_bias + tid * N);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float y = (float)x[i];
    const uint32_t c = many[i];
    if (c) {
      y = y > 0.f ? y / r : y * r;
      const uint32_t n = c & ~kSeen;
      if (n) y = y - freq * (float)n - pres;
    }
    const int at = (int)last[i];
    if (at >= 0) y += A.bias[b * A.ld_bias + at];
    if (!((word >> ((v + i) & 31)) & 1u)) y = -__builtin_inff();
    x[i] = (T)y;
  }
  T* dst = out + b * ld_o + v;
  if (whole) {
    Some<T, N> s;
#pragma unroll
    for (int i = 0; i < N; ++i) s.x[i] = x[i];
    __builtin_memcpy(dst, &s, sizeof s);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (v + i < A.V) dst[i] = x[i];
  }
}

// As few tokens a thread as give about two workgroups per CU, 8 at most: every workgroup
// reads the whole text.  (1, 4 and 8 a thread, us: one row of 32000 3.1, 3.6, 4.5; 64 rows of
// 32000, texts to 8000, 18.1, 9.4, 9.2, without texts 9.0, 4.8, 5.1; 256 rows 34, 15.6, 12.8; 64
// of 130001 51, 23.2, 21.3.)
template <class T>
int adjust(const Adjust& A, const void* logits, long ld, void* out, long ld_o, long B,
           hipStream_t stream) {
  const long wgs = B * hn_cdiv(A.V, kThreads), most = 2 * hn_device_cus();
  auto launch = [&](auto kernel, int n) {
    kernel<<<dim3(hn_cdiv(A.V, kThreads * n), B), kThreads, kThreads * n * (A.n ? 8 : 4), stream>>>(
        A, (const T*)logits, ld, (T*)out, ld_o);
  };
  if (wgs <= most) launch(adjust_kernel<T, 1>, 1);
  else if (wgs <= 4 * most) launch(adjust_kernel<T, 4>, 4);
  else launch(adjust_kernel<T, 8>, 8);
  HN_LAUNCH_CHECK("hn_adjust_logits");
  return 0;
}

}  // namespace

extern "C" int hn_adjust_logits(const void* logits, long ld, int dtype, const long* text,
                                long ld_text, long width, const long* lens, const long* first,
                                const float* repetition, const float* presence,
                                const float* frequency, float repetition1, float presence1,
                                float frequency1, const long* bias_ids, long ld_ids,
                                const float* bias, long ld_bias, long biases, const int* allowed,
                                long ld_allowed, long B, long V, void* out, long ld_out,
                                void* stream) {
  HN_ARG_CHECK(dtype >= 0 && dtype <= 2, "hn_adjust_logits: dtype %d (0 fp16, 1 bf16, 2 fp32)",
               dtype);
  HN_ARG_CHECK(B >= 0 && B < 65536 && V >= 0 && V < 1l << 31, "hn_adjust_logits: %ld rows of %ld",
               B, V);
  HN_ARG_CHECK(biases >= 0 && biases < 1l << 31 && width >= 0 && width < 1l << 31,
               "hn_adjust_logits: %ld biases, %ld tokens of text", biases, width);
  if (B == 0 || V == 0) return 0;
  HN_ARG_CHECK(logits && out && (width == 0 || text) && (biases == 0 || (bias_ids && bias)),
               "hn_adjust_logits: null operand");
  HN_ARG_CHECK(ld >= V && ld_out >= V && ld_text >= width && ld_ids >= biases &&
                   ld_bias >= biases && (!allowed || ld_allowed >= (V + 31) / 32),
               "hn_adjust_logits: rows that overlap");
  const Adjust A = {width ? text : nullptr, ld_text, width, lens, first, repetition, presence,
                    frequency, repetition1, presence1, frequency1, bias_ids, bias, ld_ids, ld_bias,
                    biases, allowed, ld_allowed, V};
  return (dtype == 0 ? adjust<h16> : dtype == 1 ? adjust<b16> : adjust<float>)(
      A, logits, ld, out, ld_out, B, (hipStream_t)stream);
}
