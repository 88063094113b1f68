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
//
// Measured: 19162 tokens of 16 + 4 heads of 128 in 7 prompts, rms norms, three
// axes, 8-bit cache, 63 us with inputs from memory (3.4 TB/s), 48 with those of the
// call before still in the memory-side cache (a 16-bit cache: 64 and 47); 96 tokens
// 6.1, one token 3.5 (loads one after another: starts, rows and page, angles'
// positions).  With rows of q, k and v mixed in a wave, sums by shuffles and angles
// at a stride of 64 floats the prompts took 96.
#include "mx8.hpp"
#include "seq_common.hpp"

namespace tx {

constexpr int NR_THREADS = 256;
// Tokens from which on workgroups of 8, not 4, still fill the card (1024 of them):
// fewer angles' rounds and starts a token.
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
// workgroup takes.  A wave takes 64 / LPR rows of one kind at a time, (token,
// head) of q, of k or of v, so that pointers, strides and what is to be done are
// the whole wave's, and one token's kinds go side by side.
template <typename T, int LPR, int TURN, int TOK>
__global__ __launch_bounds__(NR_THREADS) void norm_rotary_kernel(NormRotaryArgs a) {
  __shared__ __attribute__((aligned(16))) float cosines[TOK][128], sines[TOK][128];
  __shared__ __attribute__((aligned(16))) float meet[TURN == NR_CROSS ? NR_THREADS * 8 : 4];
  constexpr int RW = 64 / LPR;
  const int tid = threadIdx.x, lane = tid & 63, wave = seq_uni(tid >> 6);
  const SeqTile t = seq_find(a.s, 1, TOK, blockIdx.x);
  const int r0 = t.tile * TOK;
  if (r0 >= t.qn) return;
  const int n = t.qn - r0 < TOK ? t.qn - r0 : TOK;
  const int half = a.rotary >> 1, HK = a.kv_heads, hd = a.head_dim, H = a.heads;
  const int key0 = t.kvn - t.qn + r0;  // key index of the first row
  const int c = lane % LPR, d = 8 * c;  // this lane's chunk of its row
  const bool in = d < hd;
  const int nq = a.q ? n * H : 0, nk = n * HK;
  // Units of RW rows: q's, k's, v's.
  const int uq = (nq + RW - 1) / RW, uk = uq + (nk + RW - 1) / RW, units = uk + (a.k_cache ? uk - uq : 0);

  struct Row {
    int tt, h;  // token of the workgroup's, head
    bool some;
    u32x4 raw;
    int page;
  };
  // The rows of unit u, asked for one unit ahead.
  auto fetch = [&](int u, Row& w) {
    const bool q = u < uq, k = !q && u < uk;
    int i = (u - (q ? 0 : (k ? uq : uk))) * RW + lane / LPR;
    w.some = i < (q ? nq : nk);
    i = w.some ? i : 0;
    w.tt = seq_div(i, q ? a.by_heads : a.by_kv_heads);
    w.h = i - w.tt * (q ? H : HK);
    const T* p = (const T*)(q ? a.q : (k ? a.k : a.v));
    const int64_t st = q ? a.q_st : (k ? a.k_st : a.v_st), sh = q ? a.q_sh : (k ? a.k_sh : a.v_sh);
    p += (int64_t)(t.q0 + r0) * st;
    w.raw = u32x4{0, 0, 0, 0};
    if (in && w.some) w.raw = ld128(p + (w.tt * st + w.h * sh + d));
    w.page = -1;
    if (!q && a.k_cache && w.some) w.page = seq_page(a.s, t.b, key0 + w.tt);
  };
  Row w, next;
  if (wave < units) fetch(wave, w);  // in flight beside the angles

  for (int i = tid; i < n * half; i += NR_THREADS) {
    const int tt = seq_div(i, a.by_half), p = i - tt * half;
    const int axis = a.axes > 1 ? seq_cut(a.pair_axis[p], 0, a.axes - 1) : 0;
    const int64_t pos = a.positions ? a.positions[axis * a.positions_ld + t.q0 + r0 + tt] : (int64_t)(key0 + tt);
    const uint64_t phase = (uint64_t)pos * a.steps[p];
    float sn, cn;
    sincospif((float)(int64_t)phase * 0x1p-63f, &sn, &cn);
    cosines[tt][p] = cn * a.amplitude;
    sines[tt][p] = sn * a.amplitude;
  }
  __syncthreads();

  const float inv_hd = 1.0f / (float)hd;
  for (int u = wave; u < units; u += NR_THREADS / 64) {
    if (u + NR_THREADS / 64 < units) fetch(u + NR_THREADS / 64, next);
    const bool is_q = u < uq, is_v = u >= uk;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = unpack8<T>(w.raw, e);
    u32x4 out = w.raw;
    if (!is_v) {
      if (a.norm != TX_NORM_NONE) {
        if (a.norm == TX_NORM_LAYER) {
          float s = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) s += x[e];
          const float mu = nr_sum<LPR>(s) * inv_hd;
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = in ? x[e] - mu : 0.f;
        }
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += x[e] * x[e];
        const float r = rsqrtf(nr_sum<LPR>(s) * inv_hd + a.eps);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] *= r;
        const void* weight = is_q ? a.q_weight : a.k_weight;
        const void* bias = is_q ? a.q_bias : a.k_bias;
        const int at = (in ? d : 0) + w.h * a.param_sh;
        float p[8];
        if (weight) {
          nr_params<T>(weight, a.param_f32, at, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= p[e];
        }
        if (bias) {
          nr_params<T>(bias, a.param_f32, at, p);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] += p[e];
        }
      }
      // The turn.
      const float *cw = cosines[w.tt], *sw = sines[w.tt];
      if constexpr (TURN == NR_INTER) {
        const int p0 = d >> 1;
        if (d < a.rotary) {
          const f32x4 cn = *reinterpret_cast<const f32x4*>(cw + p0), sn = *reinterpret_cast<const f32x4*>(sw + p0);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = x[2 * j], q = x[2 * j + 1];
            if (d + 2 * j < a.rotary) {
              x[2 * j] = p * cn[j] - q * sn[j];
              x[2 * j + 1] = q * cn[j] + p * sn[j];
            }
          }
        }
      } else if constexpr (TURN == NR_ROW || TURN == NR_LANES) {
        const int hc = half >> 3;  // chunks of a half
        const bool first = c < hc, turns = TURN == NR_ROW || c < 2 * hc;
        const int p0 = turns ? d - (first ? 0 : half) : 0;
        const uint32_t sign = first ? 0x80000000u : 0u;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const f32x4 cn = *reinterpret_cast<const f32x4*>(cw + p0 + 4 * g), sn = *reinterpret_cast<const f32x4*>(sw + p0 + 4 * g);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float& y = x[4 * g + e];
            const float z = TURN == NR_ROW ? nr_across<LPR>(y) : __shfl(y, turns ? lane + (first ? hc : -hc) : lane, 64);
            // first half: y cos - z sin; second: y cos + z sin
            const float v = y * cn[e] + __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, z) ^ sign) * sn[e];
            y = turns ? v : y;
          }
        }
      } else {
        float* mine = meet + (tid - c) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) mine[d + e] = x[e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int at = d + e;
          if (at < a.rotary) {
            const bool first = at < half;
            const float z = mine[first ? at + half : at - half];
            const int p = first ? at : at - half;
            x[e] = first ? x[e] * cw[p] - z * sw[p] : x[e] * cw[p] + z * sw[p];
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      if (is_q || a.k_out || !a.k_scales) {
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = pack2<T>(x[2 * j], x[2 * j + 1]);
      }
      T* to = (T*)(is_q ? a.q_out : a.k_out);
      if (to && in && w.some) {
        const int64_t st = is_q ? a.qo_st : a.ko_st, sh = is_q ? a.qo_sh : a.ko_sh;
        to += (int64_t)(t.q0 + r0) * st;
        st128(to + (w.tt * st + w.h * sh + d), out);
      }
    }
    if (!is_q && a.k_cache) {
      const int slot = (key0 + w.tt) & ((1 << a.s.page_log2) - 1);
      const int64_t sp = is_v ? a.vc_sp : a.kc_sp, sh = is_v ? a.vc_sh : a.kc_sh, st = is_v ? a.vc_st : a.kc_st;
      void* cache = is_v ? a.v_cache : a.k_cache;
      if (!a.k_scales) {
        if (w.page >= 0 && in) st128((T*)cache + (w.page * sp + w.h * sh + slot * st + d), out);
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
          st64((uint8_t*)cache + (w.page * sp + w.h * sh + slot * st + d), u32x2{mx_codes(x, inv), mx_codes(x + 4, inv)});
          if ((c & 3) == 0) {
            uint8_t* s = is_v ? a.v_scales : a.k_scales;
            const int64_t ssp = is_v ? a.vs_sp : a.ks_sp, ssh = is_v ? a.vs_sh : a.ks_sh, sst = is_v ? a.vs_st : a.ks_st;
            s[w.page * ssp + w.h * ssh + slot * sst + (c >> 2)] = (uint8_t)(ex + 127);
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
