// Attention of new tokens over a paged cache of 8 bits, and of draft trees over
// one of 16 or 8 bits.
//
//   o[t, h] = sum_j p_j v_j,   p_j = exp(s_j - max s) / sum exp(s - max s),
//   s_j = scale * q[t, h] . k[j, h / group]
// over the keys that row t sees: all of its sequence up to its own (causal), or
// those before the new tokens and the new ones whose bit in t's mask row is set.
//
// One wave a row: scores of 64 keys at a time (a key a lane), running maximum and
// sum, then the keys' values one after another, two elements a lane.
#include "mx8.hpp"
#include "seq_common.hpp"

namespace tx {

template <typename T, int HD, bool MX>
__global__ __launch_bounds__(64) void cache_attention_rows_kernel(SeqAttnArgs a) {
  const float NEG_INF = -__builtin_inff();
  const SeqTile t = seq_find(a.s, 1, 1, blockIdx.x);
  if (t.tile >= t.qn) return;
  const int lane = threadIdx.x, h = blockIdx.y, hk = h / a.group, i = t.tile;
  const int64_t tok = t.q0 + i;
  const int cap = a.s.max_pages << a.s.page_log2, ps1 = (1 << a.s.page_log2) - 1;
  const int base = t.kvn - t.qn;
  const int lim = a.tree ? t.kvn : (a.causal ? base + i + 1 : t.kvn);
  auto sees = [&](int j) {
    if (j >= lim) return false;
    const int x = j - base;
    if (!a.tree || x < 0) return true;
    return x < 64 * a.tree_words && ((a.tree[tok * a.tree_ld + (x >> 6)] >> (x & 63)) & 1);
  };
  __shared__ float q[HD];
  for (int d = lane; d < HD; d += 64) q[d] = to_f32(((const T*)a.q)[tok * a.q_st + h * a.q_sh + d]);
  __syncthreads();
  auto value = [&](const void* p, const uint8_t* s, int64_t at, int64_t sat, int d) {
    if constexpr (MX) {
      const u32x4 v = mx_values<T>(((const uint8_t*)p)[at + d], 0, mx_scale(s[sat + d / MX_BLOCK]));
      return unpack8<T>(v, 0);
    } else {
      return to_f32(((const T*)p)[at + d]);
    }
  };
  float m = NEG_INF, l = 0.f, o[HD / 64];
  for (int e = 0; e < HD / 64; ++e) o[e] = 0.f;
  bool lost = false, some = false;
  for (int j0 = 0; j0 < lim; j0 += 64) {
    const int j = j0 + lane;
    bool seen = sees(j);
    some |= seen;
    const int page = seen ? seq_page(a.s, t.b, j) : 0;
    lost |= seen && (j >= cap || page < 0);
    seen = seen && page >= 0 && j < cap;
    float s = NEG_INF;
    if (seen) {
      const int64_t at = page * a.k_sp + hk * a.k_sh + (j & ps1) * a.k_st;
      const int64_t sat = page * a.ks_sp + hk * a.ks_sh + (j & ps1) * a.ks_st;
      s = 0.f;
      for (int d = 0; d < HD; ++d) s += q[d] * value(a.k, a.k_scales, at, sat, d);
      s *= a.scale;
    }
    float mx = s;
    for (int x = 32; x > 0; x >>= 1) mx = __builtin_elementwise_maximum(mx, __shfl_xor(mx, x, 64));
    const float m_new = __builtin_elementwise_maximum(m, mx);
    const float corr = m == NEG_INF ? 0.f : expf(m - m_new);
    const float p = seen && !(m_new == NEG_INF) ? expf(s - m_new) : 0.f;
    m = m_new;
    l = l * corr + wave_sum(p);
    for (int e = 0; e < HD / 64; ++e) o[e] *= corr;
    uint64_t who = __ballot(seen);
    while (who) {
      const int x = (int)__builtin_ctzll(who);
      who &= who - 1;
      const float px = __shfl(p, x, 64);
      const int64_t pg = __shfl(page, x, 64), slot = (j0 + x) & ps1;
      const int64_t at = pg * a.v_sp + hk * a.v_sh + slot * a.v_st, sat = pg * a.vs_sp + hk * a.vs_sh + slot * a.vs_st;
      for (int e = 0; e < HD / 64; ++e) o[e] += px * value(a.v, a.v_scales, at, sat, lane + 64 * e);
    }
  }
  lost = __any(lost);
  some = __any(some);
  for (int e = 0; e < HD / 64; ++e) {
    const float y = lost ? __builtin_nanf("") : (some ? o[e] / l : 0.f);
    ((T*)a.o)[tok * a.o_st + h * a.o_sh + lane + 64 * e] = from_f32<T>(y);
  }
}

template <typename T, int HD>
static int launch_hd(const SeqAttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)seq_tiles(a.s, 1, 1), (unsigned)a.heads);
  if (a.k_scales) cache_attention_rows_kernel<T, HD, true><<<grid, 64, 0, st>>>(a);
  else cache_attention_rows_kernel<T, HD, false><<<grid, 64, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
}

int launch_cache_attention(const SeqAttnArgs& a, int dt, hipStream_t st) {
  if (dt == TX_BF16) return a.head_dim == 64 ? launch_hd<bf16, 64>(a, st) : launch_hd<bf16, 128>(a, st);
  return a.head_dim == 64 ? launch_hd<f16, 64>(a, st) : launch_hd<f16, 128>(a, st);
}

}  // namespace tx
