// span_meets_blocks (csrc/limits.hpp) against a walk over the blocks' bytes.
// Prints "ok" or what failed.
#include <stdio.h>

#include "limits.hpp"

int main() {
  int fails = 0;
  for (int64_t stride = 0; stride <= 9; ++stride)
    for (int64_t extent = 1; extent <= 6; ++extent)
      for (int64_t count = 1; count <= 5; ++count)
        for (uintptr_t a = 0; a < 200; ++a)
          for (int64_t bytes = 0; bytes <= 24; ++bytes) {
            const uintptr_t b = 60;
            bool want = false;
            for (int64_t k = 0; k < count; ++k) {
              const uintptr_t lo = b + (uintptr_t)(k * stride * 2), hi = lo + (uintptr_t)(extent * 2);
              want = want || (bytes > 0 && a < hi && lo < a + (uintptr_t)bytes);
            }
            if (tx::span_meets_blocks(a, bytes, b, stride, extent, count) != want && fails++ < 10)
              printf("FAIL [%d, +%d) over %d blocks of %d at %d: not %d\n", (int)a, (int)bytes, (int)count, (int)extent,
                     (int)stride, (int)want);
          }
  // (No 64-bit product overflows.)
  if (!tx::span_meets_blocks((uintptr_t)1 << 62, 2, 0, (int64_t)1 << 40, (int64_t)1 << 40, (int64_t)1 << 30)) {
    printf("FAIL far\n");
    ++fails;
  }
  if (!fails) printf("ok\n");
  return fails != 0;
}
