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

// A row's sequence (-1: no sequence's) and position (-1: its sequence takes no part).
struct Row {
  int b;
  long pos;
};
__device__ __forceinline__ Row row_in(const Step& P, int b, int n) {
  const long C = P.lens[b];
  if (C < 0) return {b, -1};
  return {b, (C < 1l << 62 ? C : 1l << 62) + n};  // (no sum wraps)
}
// Row t, of sequence b or a later one.
__device__ __forceinline__ Row row_from(const Step& P, int t, int b) {
  while (b < P.B && P.starts[b + 1] <= t) ++b;
  if (b >= P.B || P.starts[b] > t) return {-1, -1};
  return row_in(P, b, t - P.starts[b]);
}
// Row t, by a whole wave whose first lane's row is none behind the others': the sequences
// that end at or before that row are counted by ballots, a lane goes on from there.
__device__ __forceinline__ Row row_near(const Step& P, int t) {
  if (!P.starts) return row_in(P, t, 0);
  const int lane = threadIdx.x & 63, t0 = __builtin_amdgcn_readfirstlane(t);
  int b = 0;
  for (int c = 0; c < P.B; c += 64) {
    const int at = c + lane;
    b += __popcll(__ballot(at < P.B && P.starts[at < P.B ? at + 1 : P.B] <= t0));
  }
  return row_from(P, t, b);
}

// The page of a position, -1 where the table names none.
__device__ __forceinline__ long page_of(const Step& P, int b, long pos) {
  const long col = pos >> (__builtin_ctz(P.page));
  if (col >= P.cols) return -1;
  const int id = P.table[(long)b * P.ld + col];
  return id >= 0 && id < P.pages ? id : -1;
}
