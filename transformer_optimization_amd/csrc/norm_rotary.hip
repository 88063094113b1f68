// Norms of query and key heads, rotary positions of several axes, and the
// append to a paged cache of 16 or 8 bits, one pass over q, k and v.
//
// A head x of q or k, in fp32 throughout:
//   y = (x - mu) / sqrt(mean((x - mu)^2) + eps) * weight + bias   (mu = 0: rms)
// then pair i turns by t = 2 pi p_axis(i) f_i (angles as in rotary.hip), and the
// result is rounded once: to 16 bits, or to codes and scales of blocks of 32
// (mx8.hpp).
//
// Bound by memory: 4 heads head_dim + kv_heads head_dim (4 + 2 held) bytes a
// token, held = 2 or 33/32.  A workgroup takes R tokens of one sequence, forms
// their angles once in LDS, and gives each head's row to LPR lanes of 8 elements:
// norms and block maxima are sums and maxima over a few lanes, and nothing of a
// row is read by another wave, so rows may be turned in place.
#include "mx8.hpp"
#include "seq_common.hpp"

namespace tx {

constexpr int NR_THREADS = 256;
// Tokens from which on workgroups of 8 still fill the card, for 4.
constexpr int NR_MANY = 8192;

// How the turn's pairs meet: INTER, both in one lane; ROW, in the half layout
// where a head fills its lanes and turns whole, LPR / 2 lanes apart; LANES, whole
// chunks apart; CROSS, parts of chunks (through LDS).
enum { NR_INTER, NR_ROW, NR_LANES, NR_CROSS };

// x of another lane of the row of 16 lanes (CTRL: a DPP control), on the vector ALU.
template <int CTRL> __device__ __forceinline__ float nr_dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
// Over the LPR lanes of a head: pairs, fours, eights (half mirror), sixteens (mirror).
template <int LPR> __device__ __forceinline__ float nr_sum(float x) {
  x += nr_dpp<0xB1>(x);
  x += nr_dpp<0x4E>(x);
  x += nr_dpp<0x141>(x);
  if (LPR >= 16) x += nr_dpp<0x140>(x);
  if (LPR >= 32) x += __shfl_xor(x, 16, 64);
  return x;
}
// What lies LPR / 2 lanes on, cyclically.
template <int LPR> __device__ __forceinline__ float nr_across(float x) {
  if constexpr (LPR == 16) return nr_dpp<0x128>(x);  // row_ror:8
  if constexpr (LPR == 32) return __shfl_xor(x, 16, 64);
  // 8: row_shl:4 for lanes 0 .. 3 and 8 .. 11, row_shr:4 for the others
  const int v = __builtin_bit_cast(int, x);
  const int up = __builtin_amdgcn_update_dpp(0, v, 0x104, 0xf, 0x5, false);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(up, v, 0x114, 0xf, 0xa, false));
}

// Eight gains or shifts (of the tensors' type or fp32) from element i on.
template <typename T>
__device__ __forceinline__ void nr_params(const void* p, int f32, int64_t i, float* w) {
  if (f32) {
    load4<float>((const float*)p + i, w);
    load4<float>((const float*)p + i + 4, w + 4);
  } else {
    const u32x4 x = ld128((const T*)p + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = unpack8<T>(x, e);
  }
}

// LPR lanes a row (the power of two that holds head_dim / 8); TOK: tokens a
// workgroup takes.  A head's row goes round as (token, head) of q, then of k, then
// of v, so that a wave's rows are of one kind but where kinds meet, and what only
// others need is skipped.
template <typename T, int LPR, int TURN, int TOK>
__global__ __launch_bounds__(NR_THREADS) void norm_rotary_kernel(NormRotaryArgs a) {
  __shared__ __attribute__((aligned(16))) float2 cs[TOK][128];
  __shared__ float meet[TURN == NR_CROSS ? NR_THREADS * 8 : 1];
  const int tid = threadIdx.x;
  const SeqTile t = seq_find(a.s, 1, TOK, blockIdx.x);
  const int r0 = t.tile * TOK;
  if (r0 >= t.qn) return;
  const int n = t.qn - r0 < TOK ? t.qn - r0 : TOK;
  const int half = a.rotary >> 1, HK = a.kv_heads, hd = a.head_dim, H = a.heads;
  const int key0 = t.kvn - t.qn + r0;  // key index of the first row
  const int c = tid % LPR, d = 8 * c;  // this lane's chunk of its row
  const bool in = d < hd;
  const int nq = a.q ? n * H : 0, nk = n * HK, rows = nq + nk + (a.k_cache ? nk : 0);

  // A row: its place, and what is loaded of it before the one in front is done.
  struct Row {
    int kind, tt, h;  // 0: q, 1: k, 2: v, 3: none
    u32x4 raw;
    int page;
  };
  auto fetch = [&](int i0, Row& w) {
    int i = i0 + tid / LPR;
    w.kind = i < nq ? 0 : (i < nq + nk ? 1 : (i < rows ? 2 : 3));
    i -= w.kind == 0 ? 0 : (w.kind == 1 ? nq : nq + nk);
    if (w.kind == 3) i = 0;
    w.tt = seq_div(i, w.kind == 0 ? a.by_heads : a.by_kv_heads);
    w.h = i - w.tt * (w.kind == 0 ? H : HK);
    const int64_t row = t.q0 + r0 + w.tt;
    const T* src = w.kind == 0   ? (const T*)a.q + row * a.q_st + w.h * a.q_sh
                   : w.kind == 1 ? (const T*)a.k + row * a.k_st + w.h * a.k_sh
                                 : (const T*)a.v + row * a.v_st + w.h * a.v_sh;
    w.raw = u32x4{0, 0, 0, 0};
    if (in && w.kind != 3) w.raw = ld128(src + d);
    w.page = -1;
    if (a.k_cache && (w.kind == 1 || w.kind == 2)) w.page = seq_page(a.s, t.b, key0 + w.tt);
  };
  Row w, next;
  fetch(0, w);  // in flight beside the angles

  for (int i = tid; i < n * half; i += NR_THREADS) {
    const int tt = seq_div(i, a.by_half), p = i - tt * half;
    const int axis = a.axes > 1 ? seq_cut(a.pair_axis[p], 0, a.axes - 1) : 0;
    const int64_t pos = a.positions ? a.positions[axis * a.positions_ld + t.q0 + r0 + tt] : (int64_t)(key0 + tt);
    const uint64_t phase = (uint64_t)pos * a.steps[p];
    float sn, cn;
    sincospif((float)(int64_t)phase * 0x1p-63f, &sn, &cn);
    cs[tt][p] = make_float2(cn * a.amplitude, sn * a.amplitude);
  }
  __syncthreads();

  const float inv_hd = 1.0f / (float)hd;
  // Every lane of a wave runs the same iterations: the lanes of a row meet.
  for (int i0 = 0; i0 < rows; i0 += NR_THREADS / LPR) {
    if (i0 + NR_THREADS / LPR < rows) fetch(i0 + NR_THREADS / LPR, next);
    const bool is_q = w.kind == 0, turned = w.kind < 2;
    const int64_t row = t.q0 + r0 + w.tt;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = unpack8<T>(w.raw, e);
    u32x4 out = w.raw;
    if (__any(turned)) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[e];
      if (a.norm != TX_NORM_NONE) {
        if (a.norm == TX_NORM_LAYER) {
          float s = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) s += y[e];
          const float mu = nr_sum<LPR>(s) * inv_hd;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = in ? y[e] - mu : 0.f;
        }
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += y[e] * y[e];
        const float r = 1.0f / sqrtf(nr_sum<LPR>(s) * inv_hd + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= r;
        const void* weight = is_q ? a.q_weight : a.k_weight;
        const void* bias = is_q ? a.q_bias : a.k_bias;
        float p[8];
        if (weight && in && turned) {
          nr_params<T>(weight, a.param_f32, (int64_t)w.h * a.param_sh + d, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= p[e];
        }
        if (bias && in && turned) {
          nr_params<T>(bias, a.param_f32, (int64_t)w.h * a.param_sh + d, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] += p[e];
        }
      }
      // The turn.
      const float2* angles = cs[w.tt];
      if constexpr (TURN == NR_INTER) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (d + 2 * j < a.rotary) {
            const float2 w2 = angles[(d >> 1) + j];
            const float p = y[2 * j], q = y[2 * j + 1];
            y[2 * j] = p * w2.x - q * w2.y;
            y[2 * j + 1] = q * w2.x + p * w2.y;
          }
        }
      } else if constexpr (TURN == NR_ROW) {
        const bool first = c < LPR / 2;
        const float2* mine = angles + (first ? d : d - half);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = nr_across<LPR>(y[e]);
          const float2 w2 = mine[e];
          y[e] = y[e] * w2.x + z * (first ? -w2.y : w2.y);
        }
      } else if constexpr (TURN == NR_LANES) {
        const int hc = half >> 3;  // chunks of a half
        const bool first = c < hc, turns = c < 2 * hc;
        const int from = turns ? (tid & 63) + (first ? hc : -hc) : (tid & 63);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float z = __shfl(y[e], from, 64);
          if (turns) {
            const float2 w2 = angles[d - (first ? 0 : half) + e];
            y[e] = first ? y[e] * w2.x - z * w2.y : y[e] * w2.x + z * w2.y;
          }
        }
      } else {
        float* mine = meet + (tid - c) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[d + e] = y[e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = d + e;
          if (at < a.rotary) {
            const bool first = at < half;
            const float z = mine[first ? at + half : at - half];
            const float2 w2 = angles[first ? at : at - half];
            y[e] = first ? y[e] * w2.x - z * w2.y : y[e] * w2.x + z * w2.y;
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      if (turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = y[e];
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = pack2<T>(x[2 * j], x[2 * j + 1]);
        if (in) {
          if (is_q) st128((T*)a.q_out + row * a.qo_st + w.h * a.qo_sh + d, out);
          else if (a.k_out) st128((T*)a.k_out + row * a.ko_st + w.h * a.ko_sh + d, out);
        }
      }
    }
    if (a.k_cache && __any(w.page >= 0)) {
      const bool is_v = w.kind == 2;
      const int slot = (key0 + w.tt) & ((1 << a.s.page_log2) - 1);
      if (!a.k_scales) {
        if (w.page >= 0 && in)
          st128(is_v ? (T*)a.v_cache + w.page * a.vc_sp + w.h * a.vc_sh + slot * a.vc_st + d
                     : (T*)a.k_cache + w.page * a.kc_sp + w.h * a.kc_sh + slot * a.kc_st + d, out);
      } else {
        // The block's largest magnitude, by its bits (of 32 elements: four lanes).
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t m = __builtin_bit_cast(uint32_t, x[e]) & 0x7fffffffu;
          top = m > top ? m : top;
        }
        // Infinities, NaN and what is near the end of the range take their time.
        if (__any(top > __builtin_bit_cast(uint32_t, Mx<T>::TOP))) {
          float m = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            m = fmaxf(m, mx_magnitude<T>(x[e]));
            x[e] = mx_within<T>(x[e]);
          }
          top = __builtin_bit_cast(uint32_t, m);
        }
        float m = __builtin_bit_cast(float, top);
        m = fmaxf(m, nr_dpp<0xB1>(m));
        m = fmaxf(m, nr_dpp<0x4E>(m));
        const int ex = mx_exponent<T>(m);
        const float inv = mx_power(-ex);
        if (w.page >= 0 && in) {
          uint8_t* to = is_v ? (uint8_t*)a.v_cache + w.page * a.vc_sp + w.h * a.vc_sh + slot * a.vc_st
                             : (uint8_t*)a.k_cache + w.page * a.kc_sp + w.h * a.kc_sh + slot * a.kc_st;
          st64(to + d, u32x2{mx_codes(x, inv), mx_codes(x + 4, inv)});
          if ((c & 3) == 0) {
            uint8_t* s = is_v ? a.v_scales + w.page * a.vs_sp + w.h * a.vs_sh + slot * a.vs_st
                              : a.k_scales + w.page * a.ks_sp + w.h * a.ks_sh + slot * a.ks_st;
            s[c >> 2] = (uint8_t)(ex + 127);
          }
        }
      }
    }
    w = next;
  }
}

template <typename T, int LPR, int TOK>
static int launch_lpr(const NormRotaryArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)seq_tiles(a.s, 1, TOK)), block(NR_THREADS);
  if (a.interleaved) norm_rotary_kernel<T, LPR, NR_INTER, TOK><<<grid, block, 0, st>>>(a);
  else if (a.rotary % 16) norm_rotary_kernel<T, LPR, NR_CROSS, TOK><<<grid, block, 0, st>>>(a);
  else if (a.rotary == 8 * LPR) norm_rotary_kernel<T, LPR, NR_ROW, TOK><<<grid, block, 0, st>>>(a);
  else norm_rotary_kernel<T, LPR, NR_LANES, TOK><<<grid, block, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
}

template <typename T, int TOK>
static int launch_tok(const NormRotaryArgs& a, hipStream_t st) {
  if (a.head_dim <= 64) return launch_lpr<T, 8, TOK>(a, st);
  if (a.head_dim <= 128) return launch_lpr<T, 16, TOK>(a, st);
  return launch_lpr<T, 32, TOK>(a, st);
}

template <typename T>
static int launch_typed(NormRotaryArgs a, hipStream_t st) {
  a.by_heads = seq_div_by(a.heads);
  a.by_kv_heads = seq_div_by(a.kv_heads);
  a.by_half = seq_div_by(a.rotary >> 1);
  return a.s.tokens >= NR_MANY ? launch_tok<T, 8>(a, st) : launch_tok<T, 4>(a, st);
}

int launch_norm_rotary_append(const NormRotaryArgs& a, int dt, hipStream_t st) {
  return dt == TX_BF16 ? launch_typed<bf16>(a, st) : launch_typed<f16>(a, st);
}

}  // namespace tx
