// Logits adjusted before a token is drawn from them: penalties for tokens that the
// text holds, biases, and the tokens that a grammar allows.
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

constexpr int kThreads = 256, kChunk = 2048;
constexpr uint32_t kSeen = 1u << 31;

// A workgroup takes kChunk tokens of a row.  Their counts are gathered in LDS from the
// whole text (integers, so any order gives the same), and of several biases for a
// token the last one's index.
template <class T>
__global__ __launch_bounds__(kThreads) void adjust_kernel(Adjust A, const T* logits, long ld,
                                                          T* out, long ld_o) {
  __shared__ uint32_t s_count[kChunk];
  __shared__ int s_bias[kChunk];
  const int b = blockIdx.y, tid = threadIdx.x;
  const long v0 = (long)blockIdx.x * kChunk;
  for (int i = tid; i < kChunk; i += kThreads) s_count[i] = 0, s_bias[i] = -1;
  __syncthreads();
  if (A.text) {
    long n = A.lens ? A.lens[b] : A.width;
    n = n < A.width ? n : A.width;
    const long first = A.first ? A.first[b] : 0;
    const long* text = A.text + b * A.ld_text;
    for (long i = tid; i < n; i += kThreads) {
      const unsigned long at = (unsigned long)(text[i] - v0);
      if (at >= kChunk) continue;
      if (i < first) atomicOr(&s_count[at], kSeen);
      else atomicAdd(&s_count[at], 1u);
    }
  }
  for (long i = tid; i < A.n; i += kThreads) {
    const unsigned long at = (unsigned long)(A.ids[b * A.ld_ids + i] - v0);
    if (at < kChunk) atomicMax(&s_bias[at], (int)i);
  }
  __syncthreads();
  const float r = A.rep ? A.rep[b] : A.rep1, pres = A.pres ? A.pres[b] : A.pres1;
  const float freq = A.freq ? A.freq[b] : A.freq1;
  for (int i = tid; i < kChunk && v0 + i < A.V; i += kThreads) {
    const long v = v0 + i;
    float x = (float)logits[b * ld + v];
    const uint32_t c = s_count[i];
    if (c) {
      x = x > 0.f ? x / r : x * r;
      const uint32_t n = c & ~kSeen;
      if (n) x = x - freq * (float)n - pres;
    }
    if (s_bias[i] >= 0) x += A.bias[b * A.ld_bias + s_bias[i]];
    if (A.allowed && !((A.allowed[b * A.ld_allowed + (v >> 5)] >> (v & 31)) & 1))
      x = -__builtin_inff();
    out[b * ld_o + v] = (T)x;
  }
}

template <class T>
int adjust(const Adjust& A, const void* logits, long ld, void* out, long ld_o, long B,
           hipStream_t stream) {
  adjust_kernel<T><<<dim3(hn_cdiv(A.V, kChunk), B), kThreads, 0, stream>>>(
      A, (const T*)logits, ld, (T*)out, ld_o);
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
