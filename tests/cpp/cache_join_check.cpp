// The join of a row's parts adds 32-bit byte offsets to the address of its first
// part (csrc/attention_seq.hpp): parts x K/V heads x a tile's rows x head_dim fp32
// values stay below 2^32 for every cut of a call, and parts x K/V heads within 8
// CUs' worth, by either rule (csrc/seq_cut.hpp).
// Prints "ok" or what failed.
#include <stdio.h>

#include <initializer_list>

#include "seq_cut.hpp"

using namespace tx;

int main() {
  int fails = 0;
  int64_t most = 0;
  for (int cus : {64, 256, 304})
    for (int hk : {1, 2, 3, 8, 64, 127, 128, 255, 256, 257, 511, 512, 513, 607, 608, 1024, 65535})
      for (int group : {1, 2, 16})
        for (int hd : {64, 128})
          for (int64_t tokens : {1, 8, 17, 128, 129, 4096, 1 << 20})
            for (int64_t batch : {1, 16, 1000})
              for (int64_t max_q : {(int64_t)1, tokens})
                for (int call = 0; call < 2; ++call)
                  for (int64_t rows : {(int64_t)1, (int64_t)16, (int64_t)17, (int64_t)128, tokens * group})
                    for (int keys : {256, 512, 1000, 4096, 16384, 131072, 1 << 30}) {
                      SeqShape s = seq_shape(tokens, batch, group, hk, hd, max_q, cus);
                      if (call) s.call_items = (int)seq_call_items(tokens, batch, group, hk, max_q);
                      const SeqCut c = seq_cut_of(s, (int)rows, keys);
                      if (c.parts <= 1) continue;
                      const int64_t pairs = (int64_t)c.parts * hk, n = seq_least(rows, c.tile_rows);
                      if (pairs > most) most = pairs;
                      if (pairs * n * hd * 4 < (int64_t)1 << 32 && pairs <= 8 * (int64_t)cus) continue;
                      if (++fails < 10)
                        printf("FAIL cus %d kv_heads %d group %d hd %d tokens %ld batch %ld max_q %ld call %d: %ld rows, %d "
                               "keys: %d parts\n", cus, hk, group, hd, (long)tokens, (long)batch, (long)max_q, call, (long)rows,
                               keys, c.parts);
                    }
  if (most <= 4 * 256) {  // the larger bound is reached: else what is checked is not what it says
    printf("FAIL at most %ld parts and heads\n", (long)most);
    ++fails;
  }
  if (!fails) printf("ok\n");
  return fails != 0;
}
