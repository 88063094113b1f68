// Launches of the attention over a paged 8-bit cache, and of draft trees over
// one of 16 or 8 bits: the kernels of attention_seq.hpp, whose few-row items and
// tiles form their operands from codes and scales, or hide what a row's mask does
// not name.
//
// What an 8-bit cache changes is the bytes of few rows (64 streams of 3000 to 30000
// keys: 245 us for 381 of 16 bits) and, in tiles, the way into LDS (512 tokens over
// 32768 keys: 170 us for 160 by DMA, beside which the next scores are formed).  A tree costs a compare more for keys before
// the drafts, which no mask touches, and a window of 64 mask bits for a lane's keys
// behind them.
#include "attention_seq.hpp"

namespace tx {

int64_t cache_attention_workspace(const SeqAttnArgs& a0) {
  SeqAttnArgs a = a0;
  sq_finish<SQ_PAGED | SQ_MX8>(a);
  return sq_bounds(a).partials * (a.head_dim + 2);
}

template <typename T, int HD>
static int launch_hd(const SeqAttnArgs& a, hipStream_t st) {
  if (!a.tree) return sq_launch_paged<T, HD, SQ_PAGED | SQ_MX8>(a, st);
  if (a.k_scales) return sq_launch_paged<T, HD, SQ_PAGED | SQ_MX8 | SQ_TREE>(a, st);
  return sq_launch_paged<T, HD, SQ_PAGED | SQ_TREE>(a, st);
}

int launch_cache_attention(const SeqAttnArgs& a, int dt, hipStream_t st) {
  if (dt == TX_BF16) return a.head_dim == 64 ? launch_hd<bf16, 64>(a, st) : launch_hd<bf16, 128>(a, st);
  return a.head_dim == 64 ? launch_hd<f16, 64>(a, st) : launch_hd<f16, 128>(a, st);
}

}  // namespace tx
