// How a paged attention call's work is cut into items, and what that bounds.
// Plain C++ (constexpr functions run on the host and on the device): tests
// compile this header with the host compiler.
//
// A sequence of at most SEQ_FEW rows (query heads of one K/V head x new
// tokens) is bound by reading its keys: one item per K/V head and part of the
// keys, every row in it.  More rows: tiles of 128 rows, their keys in parts
// where the tiles alone leave the card idle.  The cut of a sequence depends on
// nothing but its own rows, keys and head counts (and the card), so that its
// result does not change with the batch around it.
#pragma once

#include <stdint.h>

namespace tx {

constexpr int SEQ_FEW = 16;
constexpr int SEQ_TILE = 128;
// Keys of a part of few rows are a multiple of 256, two blocks of 32 for each of
// 4 waves (128: 32 streams of up to 2047 keys 24.5 us for 18.4; 512: 64 streams
// of 8192 keys 131 us for 141, but one of them 15.5 for 13.6).
constexpr int SEQ_PART_FEW = 256;
constexpr int SEQ_PART_TILE = 512;  // fewer are not worth writing and joining partial rows for
constexpr int SEQ_WAVE_PARTS = 16;  // rows of up to so many parts are joined by one wave
// Parts of a row at most: what the join holds, one part a thread.
constexpr int SEQ_JOIN_PARTS = 256;

struct SeqShape {
  int group, kv_heads, cus;
  // A single tile's keys are cut as one of so many tiles': of two at head dim
  // 128, where half as many parts, of twice the keys, are as fast (8192 to
  // 131072 keys, 1 to 8 K/V heads: -9% to +2%; at head dim 64 up to 35% slower)
  // and a call's partial results may be half as many.
  int least_tiles;
  int few_parts;  // most parts of few-row items
  int few;  // rows of a tile when the call has few-row items only (<= SEQ_FEW), else 0
};
struct SeqCut {
  int tiles, tile_rows;
  int parts, part_keys;  // more than one part: each row has a partial result of each
  bool few;
};
constexpr int seq_ceil(int x, int y) { return (x + (y - 1)) / y; }  // (2^30 keys in parts of 2^30 fit)
constexpr int64_t seq_least(int64_t x, int64_t y) { return x < y ? x : y; }

// max_q_len: at most tokens.
constexpr SeqShape seq_shape(int64_t tokens, int64_t batch, int group, int kv_heads, int head_dim, int64_t max_q_len,
                             int cus) {
  SeqShape s{group, kv_heads, cus, head_dim == 128 ? 2 : 1, 1, 0};
  if (cus / kv_heads > 1) s.few_parts = (int)seq_least(cus / kv_heads, SEQ_JOIN_PARTS);
  const int64_t most = max_q_len * group;
  // Calls of few-row sequences only; where their tiles could pass 32-bit
  // counts (rows beyond what max_q_len promises), the general kernel.
  if (most <= SEQ_FEW && (tokens * group / most + batch) * (kv_heads + 256) < 1 << 30) s.few = (int)most;
  return s;
}

constexpr SeqCut seq_cut_of(const SeqShape& s, int rows, int keys) {
  SeqCut c{};
  c.few = s.few > 0 || rows <= SEQ_FEW;
  c.tile_rows = c.few ? (s.few > 0 ? s.few : SEQ_FEW) : SEQ_TILE;
  c.tiles = rows <= c.tile_rows ? 1 : seq_ceil(rows, c.tile_rows);
  int most = s.few_parts, step = SEQ_PART_FEW;
  if (!c.few) {
    most = seq_ceil(2 * s.cus, (c.tiles > s.least_tiles ? c.tiles : s.least_tiles) * s.kv_heads);
    step = 64;  // a key tile
    most = most < keys / SEQ_PART_TILE ? most : keys / SEQ_PART_TILE;
    most = most < SEQ_JOIN_PARTS ? most : SEQ_JOIN_PARTS;
  }
  most = most < 1 ? 1 : most;
  c.part_keys = seq_ceil(seq_ceil(keys, most), step) * step;
  c.parts = keys > 0 ? seq_ceil(keys, c.part_keys) : 1;
  return c;
}

// Upper bounds, over all lengths that these totals allow, of a call's items, of
// its partial results (of one row and part each) and of the rows to join.  cap:
// keys of a sequence at most.
struct SeqBounds {
  int64_t items, partials, join_rows;
};
constexpr SeqBounds seq_bounds(const SeqShape& s, int64_t tokens, int64_t batch, int64_t cap) {
  const int64_t rows = tokens * s.group, hk = s.kv_heads, cus = s.cus;
  const int64_t few_parts = seq_least((cap + SEQ_PART_FEW - 1) / SEQ_PART_FEW, s.few_parts);
  const int64_t few_tiles = s.few ? rows / s.few + batch : batch;
  SeqBounds b{few_tiles * hk * few_parts, few_parts > 1 ? rows * hk * few_parts : 0, 0};
  if (!s.few) {
    const int64_t seqs = seq_least(batch, rows / (SEQ_FEW + 1));  // of more than SEQ_FEW rows
    const int64_t tiles = (rows / SEQ_TILE + seqs) * hk;
    const int64_t hl = hk * s.least_tiles;
    int64_t parts = seq_least(seq_least(cap / SEQ_PART_TILE, (2 * cus + hl - 1) / hl), SEQ_JOIN_PARTS);
    parts = parts < 1 ? 1 : parts;
    b.items += seq_least(tiles * parts, tiles + seqs * 2 * cus);
    // Rows of sequences with few and of others, each in the most parts of its
    // kind; or, where few sequences bring the others, for each of those at most
    // r hk (2 cus / (t hk) + 1) of its r <= 128 t rows.
    const int64_t few = few_parts > 1 ? few_parts : 0, tile = parts > 1 ? parts : 0;
    const int64_t few_rows = seq_least(rows, batch * SEQ_FEW);
    const int64_t either = tile >= few ? rows * tile : few_rows * few + (rows - few_rows) * tile;
    const int64_t tile_most = tile ? seqs * SEQ_TILE * 2 * cus + rows * hk : 0;
    b.partials = seq_least(either * hk, few_rows * few * hk + tile_most);
  }
  b.join_rows = b.partials > 0 ? rows * hk : 0;
  return b;
}

}  // namespace tx
