// Launches of the attention over packed prompts and over a paged 16-bit cache.
#include "attention_seq.hpp"

namespace tx {

int64_t seq_attention_workspace(const SeqAttnArgs& a0) {
  SeqAttnArgs a = a0;
  sq_finish<SQ_PAGED>(a);
  return sq_bounds(a).partials * (a.head_dim + 2);
}

template <typename T, int HD>
static int launch_hd(SeqAttnArgs a, hipStream_t st) {
  if (a.paged) return sq_launch_paged<T, HD, SQ_PAGED>(a, st);
  a.by_group = seq_div_by(a.group);
  a.by_kv_heads = seq_div_by(a.kv_heads);
  const SeqOrder o = seq_order(a.s, a.group, SQ_ROWS, (int64_t)a.s.tokens * a.kv_heads * HD * 4);
  seq_attn_packed_kernel<T, HD><<<dim3((unsigned)seq_order_grid(o, a.kv_heads)), dim3(SQ_THREADS), 0, st>>>(a, o);
  return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
}

template <typename T>
static int launch_typed(const SeqAttnArgs& a, hipStream_t st) {
  return a.head_dim == 64 ? launch_hd<T, 64>(a, st) : launch_hd<T, 128>(a, st);
}

int launch_seq_attention(const SeqAttnArgs& a, int dt, hipStream_t st) {
  return dt == TX_BF16 ? launch_typed<bf16>(a, st) : launch_typed<f16>(a, st);
}

}  // namespace tx
