// Device helpers for packed sequences and paged caches: which sequence a
// workgroup serves, and where a key lies.
#pragma once

#include "common.hpp"
#include "seq_cut.hpp"
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

// A wave-uniform value that the compiler holds in vector registers (integer
// quotients are formed there), moved to a scalar one.
__device__ __forceinline__ int seq_uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ int seq_div(int x, const SeqDiv& d) {
  return (int)((__umulhi((uint32_t)x, d.m) + (uint32_t)x) >> d.s);
}

// The sequence and tile with index w: the largest b with first_tile(b) <= w,
// found by the whole wave, 64 candidates at a time (two rounds of loads up to
// 4096 sequences).  Wave-uniform; every lane takes part.  Starts that do not
// ascend give some sequence, whose bounds are cut to the tensors all the same.
__device__ __forceinline__ SeqTile seq_find(const SeqArgs& s, int group, int r, int64_t w) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = s.batch;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    const int i = lo + lane * step;
    bool below = false;
    if (lane * step < n) below = (int64_t)seq_cut(s.cu[i], 0, s.tokens) * group / r + i <= w;
    const int c = __builtin_popcountll(__ballot(below));
    const int skip = c > 0 ? (c - 1) * step : 0;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  SeqTile t;
  t.b = __builtin_amdgcn_readfirstlane(lo);
  const int q0 = seq_uni(seq_cut(s.cu[t.b], 0, s.tokens));
  const int q1 = seq_uni(seq_cut(s.cu[t.b + 1], q0, s.tokens));
  t.q0 = q0;
  t.qn = q1 - q0;
  t.kvn = s.kv_lens ? seq_uni(s.kv_lens[t.b]) : t.qn;
  t.kvn = t.kvn < 0 ? 0 : t.kvn;
  const int64_t d = w - ((int64_t)q0 * group / r + t.b);
  t.tile = (int)d;
  if (d < 0) t.qn = t.tile = 0;  // before the first sequence
  return t;
}

// Sum over the wave (all lanes active), on the vector ALU alone.
__device__ __forceinline__ int seq_wave_sum(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return __builtin_amdgcn_readlane(x, 63);
}

// Order of a call of packed prompts: the tiles of all sequences and heads in
// descending order of their index, so that under a causal mask those with the
// most keys start first, whichever sequence they belong to (16 prompts of up
// to 1021 tokens 47 -> 40 us).  Where the keys and values are more than the
// 256 MB of the memory-side cache, bands of 16 neighbouring tiles of one
// (sequence, K/V head), which read the same keys in step, are ordered instead,
// each on one XCD (workgroup i runs on XCD i % 8), whose L2 then serves them: 8
// x 16384 tokens, 16 heads with keys of their own, 10.1 -> 8.2 ms, 8 x 8192
// 2.50 -> 2.18; below that size the coarser order costs more than it saves (8 x
// 2048 156 -> 164 us).
struct SeqOrder {
  int band;   // log2 tiles of a band
  int bands;  // bound on a head's bands over all sequences
};
// More than 64 sequences keep seq_find's order (reversed), where the tail of
// one long sequence weighs little.
inline SeqOrder seq_order(const SeqArgs& s, int group, int r, int64_t kv_bytes) {
  const int64_t tiles = seq_tiles(s, group, r);
  SeqOrder o;
  o.band = s.batch <= 64 && kv_bytes >= (int64_t)1 << 28 && tiles / s.batch >= 16 ? 4 : 0;
  o.bands = (int)(s.batch > 64 ? tiles : (tiles >> o.band) + s.batch);
  return o;
}
inline int64_t seq_order_grid(const SeqOrder& o, int kv_heads) {
  return (((int64_t)o.bands * kv_heads + 7) / 8 * 8) << o.band;
}
// The tile and K/V head of workgroup wg; qn = 0: none.
__device__ __forceinline__ SeqTile seq_ordered(const SeqArgs& s, int group, int r, SeqOrder o, int kv_heads, int wg,
                                               int& hk) {
  const int i = wg >> 3, sub = i & ((1 << o.band) - 1);
  const int slot = (i >> o.band) * 8 + (wg & 7);
  const int w = seq_uni(slot / kv_heads);
  hk = slot - w * kv_heads;
  SeqTile t{};
  if (s.batch > 64) return w < o.bands ? seq_find(s, group, r, o.bands - 1 - w) : t;
  // One lane a sequence, one round of loads.
  const int lane = threadIdx.x & 63;
  const int b = lane < s.batch ? lane : s.batch - 1;
  const int q0 = seq_cut(s.cu[b], 0, s.tokens);
  const int qn = lane < s.batch ? max(seq_cut(s.cu[b + 1], 0, s.tokens) - q0, 0) : 0;
  const int n = (qn * group + r - 1) / r, nb = (n + (1 << o.band) - 1) >> o.band;
  // count(x): bands of index x or more.  count(lo) > w >= count(hi).
  auto count = [&](int x) { return seq_wave_sum(max(nb - x, 0)); };
  int lo = 0, hi = o.bands, after = 0;
  if (count(0) <= w) return t;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, c = count(mid);
    if (c > w) lo = mid;
    else {
      hi = mid;
      after = c;
    }
  }
  // The (w - count(lo + 1))-th sequence of those with a band lo.
  uint64_t has = __ballot(nb > lo);
  for (int k = w - after; k > 0; --k) has &= has - 1;
  t.b = seq_uni((int)__builtin_ctzll(has));
  t.tile = (lo << o.band) + (1 << o.band) - 1 - sub;
  t.q0 = __builtin_amdgcn_readlane(q0, t.b);
  t.qn = t.tile < __builtin_amdgcn_readlane(n, t.b) ? __builtin_amdgcn_readlane(qn, t.b) : 0;
  t.kvn = t.qn;
  return t;
}

// ---- the items of a paged call (seq_cut.hpp) ------------------------------
// A sequence of a paged call: its cut, its first item and its first partial
// result, both counted over the call.
struct SeqWork {
  int b, q0, qn, kvn;
  SeqCut cut;
  int item, partial;
};

// Walks the items of a call in ascending order, 64 sequences at a time (lane
// i: sequence base + i).  Every wave of the workgroup walks the same items and
// every lane takes part.  What the lanes hold of their sequences stays in LDS
// between the items, whose own work needs the registers: one copy, which each
// wave writes alike between two barriers.
struct SeqWalk {
  struct Lane {
    int n_items, n_partials;    // of this lane's sequence
    int at_item, at_partial;    // behind its last item and partial result (from base on)
    int q0, qn, kvn;
    int tiles, parts, part_keys;
  };
  static constexpr int LDS_INTS = 64 * 10;
  int base, items, partials;  // before sequence base
  int row;                 // first row that sequence base may hold
  int* lds;                // LDS_INTS of the workgroup

  __device__ __forceinline__ void load(const SeqArgs& s, const SeqShape& sh, bool join) {
    const int lane = threadIdx.x & 63, b = base + lane;
    const bool in = b < s.batch;
    Lane x;
    // Starts that do not ascend are raised to the largest before them, so that
    // no row is in two sequences and the host's bounds on items and units hold
    // whatever the array says.
    x.q0 = max(in ? seq_cut(s.cu[b], 0, s.tokens) : 0, row);
    const int end = in ? seq_cut(s.cu[b + 1], 0, s.tokens) : 0;
    x.kvn = in ? max(s.kv_lens[b], 0) : 0;
    const int n = min(s.batch - base, 64);  // the scans need log2(n) steps
    for (int o = 1; o < n; o <<= 1) x.q0 = max(x.q0, __shfl_up(x.q0, o, 64));  // (lanes below o see themselves)
    x.qn = max(end - x.q0, 0);
    x.n_items = x.n_partials = x.tiles = x.parts = x.part_keys = 0;
    if (x.qn > 0) {
      const SeqCut c = seq_cut_of(sh, x.qn * sh.group, min(x.kvn, s.max_pages << s.page_log2));
      x.n_items = c.tiles * c.parts * sh.kv_heads;
      x.n_partials = c.parts > 1 ? x.qn * sh.group * sh.kv_heads * c.parts : 0;
      x.tiles = c.tiles;
      x.parts = c.parts;
      x.part_keys = c.part_keys;
      if (join) {  // rows, four to an item where a wave joins one
        const int all = x.qn * sh.group * sh.kv_heads;
        x.n_items = c.parts <= 1 ? 0 : (c.parts <= SEQ_WAVE_PARTS ? seq_ceil(all, 4) : all);
      }
    }
    x.at_item = x.n_items;
    x.at_partial = x.n_partials;
    for (int o = 1; o < n; o <<= 1) {
      const int i = __shfl_up(x.at_item, o, 64), u = __shfl_up(x.at_partial, o, 64);
      if (lane >= o) {
        x.at_item += i;
        x.at_partial += u;
      }
    }
    __syncthreads();  // nobody reads the sequences before these any more
    const int f[10] = {x.n_items, x.n_partials, x.at_item, x.at_partial, x.q0, x.qn, x.kvn, x.tiles, x.parts, x.part_keys};
#pragma unroll
    for (int i = 0; i < 10; ++i) lds[64 * i + lane] = f[i];
    __syncthreads();
  }
  __device__ __forceinline__ void init(const SeqArgs& s, const SeqShape& sh, bool join, int* lds_) {
    base = items = partials = row = 0;
    lds = lds_;
    load(s, sh, join);
  }
  // Field f of the Lane of sequence base + i.
  __device__ __forceinline__ int field(int f, int i) const { return seq_uni(lds[64 * f + i]); }
  // The sequence of item w (ascending from call to call); false: past the end.
  __device__ __forceinline__ bool find(const SeqArgs& s, const SeqShape& sh, bool join, int w, SeqWork& r) {
    for (;;) {
      const int last = min(s.batch - base, 64) - 1;
      const int in_items = field(2, last);
      if (w - items < in_items) break;
      if (base + 64 >= s.batch) return false;
      items += in_items;
      partials += field(3, last);
      row = field(4, last) + field(5, last);
      base += 64;
      load(s, sh, join);
    }
    // Lanes that end before w (those past the batch do not count).
    const int lane = threadIdx.x & 63;
    const int i = __builtin_popcountll(__ballot(base + lane < s.batch && lds[64 * 2 + lane] <= w - items));
    r.b = base + i;
    r.q0 = field(4, i);
    r.qn = field(5, i);
    r.kvn = field(6, i);
    r.item = items + field(2, i) - field(0, i);
    r.partial = partials + field(3, i) - field(1, i);
    r.cut.few = sh.few > 0 || r.qn * sh.group <= SEQ_FEW;
    r.cut.tile_rows = r.cut.few ? (sh.few > 0 ? sh.few : SEQ_FEW) : SEQ_TILE;
    r.cut.tiles = field(7, i);
    r.cut.parts = field(8, i);
    r.cut.part_keys = field(9, i);
    return true;
  }
};

// The page of key j of sequence b, or -1.
__device__ __forceinline__ int seq_page(const SeqArgs& s, int b, int j) {
  const int i = j >> s.page_log2;
  if (j < 0 || i >= s.max_pages) return -1;
  const int p = s.table[(int64_t)b * s.table_ld + i];
  return (p >= 0 && p < s.num_pages) ? p : -1;
}

}  // namespace tx
