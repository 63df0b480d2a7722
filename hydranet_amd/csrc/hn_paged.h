// What a step over a paged KV cache is to its kernels (hn_paged.hip).
#pragma once
#include "hn_common.h"

typedef __bf16 b16;

struct Step {
  const int* table;  // [B][ld], cols of them valid
  long ld, cols, pages;
  const long* lens;
  const int* starts;  // [B + 1] or null: row b is sequence b's
  int B, T, nkv, page;
};

// Row t's sequence (-1: no sequence's) and position (-1: its sequence takes no part).
// By a whole wave: the sequences that end at or before t are counted by ballots.
struct Row {
  int b;
  long pos;
};
__device__ __forceinline__ Row row_of(const Step& P, int t) {
  int b = t, first = t;
  if (P.starts) {
    b = 0;
    for (int c = threadIdx.x & 63; c - (int)(threadIdx.x & 63) < P.B; c += 64)
      b += __popcll(__ballot(c < P.B && P.starts[c < P.B ? c + 1 : P.B] <= t));
    if (b >= P.B || (first = P.starts[b]) > t) return {-1, -1};
  }
  const long C = P.lens[b];
  if (C < 0) return {b, -1};
  return {b, (C < 1l << 62 ? C : 1l << 62) + (t - first)};  // (no sum wraps)
}

// The page of a position, -1 where the table names none.
__device__ __forceinline__ long page_of(const Step& P, int b, long pos) {
  const long col = pos >> (__builtin_ctz(P.page));
  if (col >= P.cols) return -1;
  const int id = P.table[(long)b * P.ld + col];
  return id >= 0 && id < P.pages ? id : -1;
}
