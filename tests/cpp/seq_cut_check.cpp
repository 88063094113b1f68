// The cut of a paged attention call (csrc/seq_cut.hpp): every row and key in
// one item, never more parts than the join holds, and the host's bounds on
// items, partial results and rows to join kept by every split of the totals, and
// of a reasonable size for ordinary calls.
// Prints "ok" or what failed.
#include <stdio.h>

#include <initializer_list>

#include "seq_cut.hpp"

using namespace tx;

static int fails = 0;
static uint64_t rng_state = 1;
static uint64_t rng() {  // splitmix64
  uint64_t z = (rng_state += 0x9E3779B97F4A7C15ull);
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
static int64_t below(int64_t n) { return (int64_t)(rng() % (uint64_t)n); }

static void check_cut(const SeqShape& s, int rows, int keys) {
  const SeqCut c = seq_cut_of(s, rows, keys);
  const int tile = c.tile_rows;
  bool ok = c.parts >= 1 && c.parts <= SEQ_JOIN_PARTS;
  ok = ok && (int64_t)c.tiles * tile >= rows && (int64_t)(c.tiles - 1) * tile < rows;
  if (keys > 0)
    ok = ok && c.part_keys % 64 == 0 && (int64_t)c.parts * c.part_keys >= keys &&
         (int64_t)(c.parts - 1) * c.part_keys < keys;
  if (!ok) {
    printf("FAIL group %d kv_heads %d cus %d few %d: %d rows, %d keys: %d tiles, %d parts of %d\n", s.group, s.kv_heads,
           s.cus, s.few, rows, keys, c.tiles, c.parts, c.part_keys);
    ++fails;
  }
}

int main() {
  const int rows_at[] = {1, 2, 15, 16, 17, 24, 31, 32, 33, 64, 127, 128, 129, 255, 256, 257, 1000, 4096, 100000, 1 << 22};
  const int keys_at[] = {0, 1, 63, 64, 255, 256, 257, 511, 512, 513, 1024, 20011, 65536, 131071, 131072, 131584, 147456,
                         200000, 262144, 300001, 1 << 20, (1 << 30) - 1, 1 << 30};
  for (int cus : {64, 256, 304})
    for (int hk : {1, 2, 3, 4, 8, 16, 64, 300, 65535})
      for (int few : {0, 1, 4, 16})
        for (int rows : rows_at)
          for (int keys : keys_at) {
            for (int hd : {64, 128}) check_cut(seq_shape(1 << 20, 1, 1, hk, hd, few ? few : 1 << 20, cus), rows, keys);
          }
  // Split totals over the sequences at random; the calls' actual work.
  for (int trial = 0; trial < 20000 && fails < 10; ++trial) {
    const int group = 1 + (int)below(16), hk = 1 + (int)below(trial % 3 ? 8 : 80), batch = 1 + (int)below(40);
    const int64_t cap = (int64_t)8 << below(20);
    const int64_t tokens = 1 + below(trial % 2 ? 64 : 3000);
    const int64_t max_q = trial % 4 == 0 ? tokens : 1 + below(tokens);  // may be too small
    const SeqShape s = seq_shape(tokens, batch, group, hk, trial % 7 ? 128 : 64, max_q, 256);
    const SeqBounds b = seq_bounds(s, tokens, batch, cap);
    int64_t left = tokens, items = 0, partials = 0, joins = 0;
    for (int i = 0; i < batch; ++i) {
      const int64_t most = trial % 5 == 0 ? (128 / group > 0 ? 128 / group : 1) : left;
      const int64_t n = i + 1 == batch && trial % 2 ? left : below((most < left ? most : left) + 1);
      left -= n;
      if (n == 0) continue;
      const int rows = (int)n * group, keys = (int)(trial % 3 ? cap : below(cap + 1));
      check_cut(s, rows, keys);
      const SeqCut c = seq_cut_of(s, rows, keys);
      items += (int64_t)c.tiles * c.parts * hk;
      if (c.parts > 1) partials += (int64_t)rows * hk * c.parts;
      if (c.parts > 1) joins += c.parts <= SEQ_WAVE_PARTS ? (rows * hk + 3) / 4 : rows * hk;
    }
    if (items > b.items || partials > b.partials || joins > b.join_rows) {
      printf("FAIL group %d kv_heads %d batch %d tokens %ld cap %ld max_q %ld: items %ld of %ld, partials %ld of %ld, joins "
             "%ld of %ld\n", group, hk, batch, (long)tokens, (long)cap, (long)max_q, (long)items, (long)b.items,
             (long)partials, (long)b.partials, (long)joins, (long)b.join_rows);
      ++fails;
    }
  }
  // Partial results of head_dim + 2 floats of calls as servers make them: one
  // chunk of 512 tokens among single ones, and those alone (without max_q_len).
  const struct {
    int64_t tokens, batch;
    int heads, hk;
    int64_t cap, max_q, mib;
  } calls[] = {{768, 257, 16, 4, 131072, 512, 400}, {576, 65, 16, 4, 32768, 512, 300}, {576, 65, 32, 8, 131072, 512, 300},
               {768, 257, 64, 8, 131072, 512, 800}, {535, 24, 16, 2, 8192, 512, 80},   {64, 64, 16, 4, 32768, 64, 33},
               {64, 64, 16, 4, 32768, 1, 33},       {512, 1, 16, 4, 32768, 512, 40}};
  for (const auto& c : calls) {
    const SeqShape s = seq_shape(c.tokens, c.batch, c.heads / c.hk, c.hk, 128, c.max_q, 256);
    const int64_t mib = (seq_bounds(s, c.tokens, c.batch, c.cap).partials * 130 * 4) >> 20;
    if (mib > c.mib) {
      printf("FAIL %ld tokens of %ld sequences, %d/%d heads, %ld keys: %ld MiB of workspace\n", (long)c.tokens,
             (long)c.batch, c.heads, c.hk, (long)c.cap, (long)mib);
      ++fails;
    }
  }
  if (!fails) printf("ok\n");
  return fails != 0;
}
