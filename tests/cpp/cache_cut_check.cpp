// The cut of a paged call whose totals cut the keys of tiles (8-bit caches, draft
// trees; csrc/seq_cut.hpp): every row and key in one item, the host's bounds on
// items, partial results and rows to join kept by every split of the totals, also
// where the longest sequence is longer than it was said to be, and counts that
// stay within 32 bits.
// Prints "ok" or what failed.
#include <stdio.h>

#include <initializer_list>

#include "seq_cut.hpp"

using namespace tx;

static int fails = 0;
static uint64_t rng_state = 7;
static uint64_t rng() {  // splitmix64
  uint64_t z = (rng_state += 0x9E3779B97F4A7C15ull);
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
static int64_t below(int64_t n) { return (int64_t)(rng() % (uint64_t)n); }

static SeqShape shape(int64_t tokens, int64_t batch, int group, int hk, int hd, int64_t max_q, int cus) {
  SeqShape s = seq_shape(tokens, batch, group, hk, hd, max_q, cus);
  s.call_items = (int)seq_call_items(tokens, batch, group, hk, max_q);
  return s;
}
static void check_cut(const SeqShape& s, int rows, int keys) {
  const SeqCut c = seq_cut_of(s, rows, keys);
  bool ok = s.call_items >= 1 && c.parts >= 1 && c.parts <= SEQ_JOIN_PARTS;
  ok = ok && (int64_t)c.tiles * c.tile_rows >= rows && (int64_t)(c.tiles - 1) * c.tile_rows < rows;
  if (keys > 0)
    ok = ok && c.part_keys % 64 == 0 && (int64_t)c.parts * c.part_keys >= keys &&
         (int64_t)(c.parts - 1) * c.part_keys < keys;
  if (!ok) {
    printf("FAIL items %d kv_heads %d: %d rows, %d keys: %d tiles, %d parts of %d\n", s.call_items, s.kv_heads, rows, keys,
           c.tiles, c.parts, c.part_keys);
    ++fails;
  }
}

int main() {
  const int keys_at[] = {0, 1, 63, 64, 127, 128, 255, 256, 300, 1000, 2048, 4095, 4096, 20011, 131072, 1 << 20, 1 << 30};
  for (int cus : {64, 256, 304})
    for (int hk : {1, 3, 8, 64, 65535})
      for (int64_t tokens : {1, 17, 64, 300, 4096, 1 << 20})
        for (int64_t batch : {1, 16, 1000})
          for (int64_t max_q : {(int64_t)1, (tokens + 1) / 2, tokens})
            for (int keys : keys_at) {
              const SeqShape s = shape(tokens, batch, 2, hk, 128, max_q, cus);
              check_cut(s, 17, keys);
              check_cut(s, (int)(2 * tokens), keys);
              // more keys are never cut into fewer parts than the bound says
              int64_t before = 0;
              for (int k = 0; k <= 1 << 15; k += 1000) {
                const int64_t p = seq_call_parts(cus, s.call_items, k);
                if (p < before) {
                  printf("FAIL cus %d items %d keys %d: %ld parts after %ld\n", cus, s.call_items, k, (long)p, (long)before);
                  ++fails;
                }
                before = p;
              }
            }
  for (int trial = 0; trial < 20000 && fails < 10; ++trial) {
    const int group = 1 + (int)below(16), hk = 1 + (int)below(trial % 3 ? 8 : 80), batch = 1 + (int)below(40);
    const int64_t cap = (int64_t)8 << below(20);
    const int64_t tokens = 1 + below(trial % 2 ? 200 : 5000);
    const int64_t max_q = trial % 4 == 0 ? tokens : 1 + below(tokens);  // may be too small
    const SeqShape s = shape(tokens, batch, group, hk, trial % 7 ? 128 : 64, max_q, 256);
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
  // The largest calls that the entry points let through and whose workspace fits
  // a card (288 GB): 32-bit counts.
  for (int hk : {1, 8, 64, 1024})
    for (int64_t tokens : {1 << 10, 1 << 16, 1 << 20, 1 << 24})
      for (int64_t batch : {1, 1000, 1 << 13})
        for (int64_t max_q : {(int64_t)1, (int64_t)64, tokens}) {
          const int64_t heads = ((int64_t)1 << 26) / tokens / hk * hk;
          if (heads < hk || heads > 65535 || batch * hk > 1 << 23) continue;
          const SeqShape s = shape(tokens, batch, (int)(heads / hk), hk, 128, max_q, 256);
          const SeqBounds b = seq_bounds(s, tokens, batch, 1 << 30);
          if (b.partials > 288000000000 / (130 * 4)) continue;
          if (b.items >= (int64_t)1 << 31 || b.partials >= (int64_t)1 << 31) {
            printf("FAIL tokens %ld batch %ld heads %ld / %d max_q %ld: items %ld partials %ld\n", (long)tokens, (long)batch,
                   (long)heads, hk, (long)max_q, (long)b.items, (long)b.partials);
            ++fails;
          }
        }
  if (!fails) printf("ok\n");
  return fails != 0;
}
