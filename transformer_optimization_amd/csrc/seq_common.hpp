// Device helpers for packed sequences and paged caches: which sequence a
// workgroup serves, and where a key lies.
#pragma once

#include "common.hpp"
#include "tx_internal.hpp"

namespace tx {

// Rows of a sequence are cut into tiles of R; row r is (token r / group, query
// head r % group of a K/V head).  Sequence b's tiles get the indices from
// first_tile(b) = cu[b] * group / R + b on: strictly ascending in b, and far
// enough apart for ceil(rows / R) tiles of each (floor(x + n) >= floor(x) +
// floor(n)), so that no prefix sum over the lengths is needed.  A grid of
// seq_tiles() covers them all; at most one tile per sequence is empty.
inline int64_t seq_tiles(const SeqArgs& s, int group, int r) {
  return (int64_t)s.tokens * group / r + s.batch;
}

struct SeqTile {
  int b;       // sequence
  int tile;    // tile within it
  int q0, qn;  // its rows in the packed tensors
  int kvn;     // its keys (may be more than the table holds)
};

__device__ __forceinline__ int seq_cut(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// The sequence and tile with index w: the largest b with first_tile(b) <= w,
// found by the whole wave, 64 candidates at a time (two rounds of loads up to
// 4096 sequences).  Wave-uniform; every lane takes part.
__device__ __forceinline__ SeqTile seq_find(const SeqArgs& s, int group, int r, int64_t w) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = s.batch;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int i = lo + lane * step;
    bool below = false;
    if (lane * step < n) below = (int64_t)seq_cut(s.cu[i], 0, s.tokens) * group / r + i <= w;
    const int c = __builtin_popcountll(__ballot(below));  // 0: not found before lo (cannot be for lo = 0)
    const int skip = c > 0 ? (c - 1) * step : 0;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  SeqTile t;
  t.b = __builtin_amdgcn_readfirstlane(lo);
  const int q0 = __builtin_amdgcn_readfirstlane(seq_cut(s.cu[t.b], 0, s.tokens));
  const int q1 = __builtin_amdgcn_readfirstlane(seq_cut(s.cu[t.b + 1], q0, s.tokens));
  t.q0 = q0;
  t.qn = q1 - q0;
  t.kvn = s.kv_lens ? __builtin_amdgcn_readfirstlane(s.kv_lens[t.b]) : t.qn;
  t.kvn = t.kvn < 0 ? 0 : t.kvn;
  const int64_t d = w - ((int64_t)q0 * group / r + t.b);
  t.tile = (int)d;
  if (d < 0) t.qn = t.tile = 0;  // before the first sequence
  return t;
}

// The page of key j of sequence b, or -1.
__device__ __forceinline__ int seq_page(const SeqArgs& s, int b, int j) {
  const int i = j >> s.page_log2;
  if (j < 0 || i >= s.max_pages) return -1;
  const int p = s.table[(int64_t)b * s.table_ld + i];
  return (p >= 0 && p < s.num_pages) ? p : -1;
}

}  // namespace tx
