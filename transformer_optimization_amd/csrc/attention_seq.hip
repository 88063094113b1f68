// Attention over packed sequences and over a paged cache, with grouped heads.
//
//   o[t, h] = sum_j p_j v_j,   p_j = exp(s_j - max s) / sum exp(s - max s),
//   s_j = scale * q[t, h] . k[j, h / group]
#include "seq_common.hpp"

namespace tx {

// Row and key addresses of one (sequence, K/V head).
template <typename T, bool PAGED>
struct SeqHead {
  const T* k;  // row 0 of the sequence, or page 0 of the cache
  const T* v;
  int b;
  __device__ __forceinline__ void init(const SeqAttnArgs& a, const SeqTile& t, int hk) {
    k = (const T*)a.k + hk * a.k_sh + (PAGED ? 0 : (int64_t)t.q0 * a.k_st);
    v = (const T*)a.v + hk * a.v_sh + (PAGED ? 0 : (int64_t)t.q0 * a.v_st);
    b = t.b;
  }
  // Offset of key j's row in units of (page, slot); false: it has no page.
  __device__ __forceinline__ bool at(const SeqAttnArgs& a, int j, const T*& kr, const T*& vr) const {
    if constexpr (PAGED) {
      const int page = seq_page(a.s, b, j), slot = j & ((1 << a.s.page_log2) - 1);
      const int pg = page < 0 ? 0 : page;
      kr = k + pg * a.k_sp + slot * a.k_st;
      vr = v + pg * a.v_sp + slot * a.v_st;
      return page >= 0;
    } else {
      kr = k + (int64_t)j * a.k_st;
      vr = v + (int64_t)j * a.v_st;
      return true;
    }
  }
};

// One query row over the keys [j0, j1), by one wave, on the vector ALU: the
// maximum and sum of the softmax first, then the weighted values, key by key.
// lane: dims lane, lane + 64, ... of o (fp32, normalised; 0 without keys).
// Every masked key is skipped, never multiplied by 0.
template <typename T, int HD, bool PAGED>
__device__ void seq_row(const SeqAttnArgs& a, const SeqHead<T, PAGED>& hp, const T* qrow, int j0, int j1,
                        float* o, float& m, float& l) {
  constexpr int DPL = HD / 64;
  const int lane = threadIdx.x & 63;
  const float NEG_INF = -__builtin_inff(), NAN_ = __builtin_nanf("");
  auto score = [&](int j, const T*& vr) {
    const T* kr;
    if (!hp.at(a, j, kr, vr)) return NAN_;  // a key that has no page
    float s = 0.f;
    for (int d = 0; d < HD; d += 8) {
      const u32x4 x = ld128(qrow + d), y = ld128(kr + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += unpack8<T>(x, e) * unpack8<T>(y, e);
    }
    return s * a.scale;
  };
  for (int i = 0; i < DPL; ++i) o[i] = 0.f;
  m = NEG_INF;
  l = 0.f;
  if (j1 <= j0) return;
  const T* vr;
  for (int j = j0 + lane; j < j1; j += 64) {
    const float s = score(j, vr), mn = fmaxf(m, s);
    l = (m == NEG_INF ? l : l * expf(m - mn)) + (mn == NEG_INF ? 0.f : expf(s - mn));
    m = mn;
    if (!(s == s)) l = NAN_;
  }
  float mw = m;
  for (int x = 32; x > 0; x >>= 1) mw = fmaxf(mw, __shfl_xor(mw, x, 64));
  l = wave_sum(m == NEG_INF ? l : l * expf(m - mw));
  m = mw;
  const float inv = 1.0f / l;  // l = 0 (every score -inf): 0 * inf below is NaN, as softmax gives
  for (int b0 = j0; b0 < j1; b0 += 64) {
    const int j = b0 + lane;
    float p = 0.f;
    if (j < j1) p = (m == NEG_INF ? 0.f : expf(score(j, vr) - m)) * inv;
    const int n = j1 - b0 < 64 ? j1 - b0 : 64;
    for (int i = 0; i < n; ++i) {
      const float pi = __shfl(p, i, 64);
      const T* kr;
      const T* vi;
      hp.at(a, b0 + i, kr, vi);
      for (int e = 0; e < DPL; ++e) o[e] += pi * to_f32(vi[lane + 64 * e]);
    }
  }
}

// One wave per (token, query head).
template <typename T, int HD, bool PAGED>
__global__ __launch_bounds__(256) void seq_attn_rows_kernel(SeqAttnArgs a) {
  const SeqTile t = seq_find(a.s, a.group, 4, blockIdx.x);
  const int hk = blockIdx.y, row = t.tile * 4 + (int)(threadIdx.x >> 6);
  if (row >= t.qn * a.group) return;
  const int i = row / a.group, h = hk * a.group + row - i * a.group;
  SeqHead<T, PAGED> hp;
  hp.init(a, t, hk);
  const int lim = a.causal ? t.kvn - t.qn + i + 1 : t.kvn;
  const int64_t tok = t.q0 + i;
  float o[HD / 64], m, l;
  seq_row<T, HD, PAGED>(a, hp, (const T*)a.q + tok * a.q_st + h * a.q_sh, 0, lim, o, m, l);
  T* orow = (T*)a.o + tok * a.o_st + h * a.o_sh;
  for (int e = 0; e < HD / 64; ++e) orow[(threadIdx.x & 63) + 64 * e] = from_f32<T>(o[e]);
}

template <typename T, int HD>
static int launch_hd(const SeqAttnArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)seq_tiles(a.s, a.group, 4), (unsigned)a.kv_heads), block(256);
  if (a.paged) seq_attn_rows_kernel<T, HD, true><<<grid, block, 0, st>>>(a);
  else seq_attn_rows_kernel<T, HD, false><<<grid, block, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
}

template <typename T>
static int launch_typed(const SeqAttnArgs& a, hipStream_t st) {
  return a.head_dim == 64 ? launch_hd<T, 64>(a, st) : launch_hd<T, 128>(a, st);
}

int64_t seq_attention_workspace(const SeqAttnArgs&) { return 0; }

int launch_seq_attention(const SeqAttnArgs& a, int dt, hipStream_t st) {
  return dt == TX_BF16 ? launch_typed<bf16>(a, st) : launch_typed<f16>(a, st);
}

}  // namespace tx
