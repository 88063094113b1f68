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
constexpr int NR_TOKENS = 4;

template <int LPR> __device__ __forceinline__ float nr_sum(float x) {
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
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

// LPR lanes a row (the power of two that holds head_dim / 8); CROSS: pairs of
// the half layout that do not lie in whole chunks meet in LDS.
template <typename T, int LPR, bool CROSS>
__global__ __launch_bounds__(NR_THREADS) void norm_rotary_kernel(NormRotaryArgs a) {
  __shared__ float2 cs[NR_TOKENS][128];
  __shared__ float meet[CROSS ? NR_THREADS * 8 : 1];
  const int tid = threadIdx.x;
  const SeqTile t = seq_find(a.s, 1, NR_TOKENS, blockIdx.x);
  const int r0 = t.tile * NR_TOKENS;
  if (r0 >= t.qn) return;
  const int n = t.qn - r0 < NR_TOKENS ? t.qn - r0 : NR_TOKENS;
  const int half = a.rotary >> 1, HK = a.kv_heads, hd = a.head_dim;
  const int key0 = t.kvn - t.qn + r0;  // key index of the first row

  for (int i = tid; i < n * half; i += NR_THREADS) {
    const int tt = i / half, p = i - tt * half;
    int axis = a.pair_axis ? a.pair_axis[p] : 0;
    axis = seq_cut(axis, 0, a.axes - 1);
    const int64_t pos = a.positions ? a.positions[axis * a.positions_ld + t.q0 + r0 + tt] : (int64_t)(key0 + tt);
    const uint64_t phase = (uint64_t)pos * a.steps[p];
    float sn, cn;
    sincospif((float)(int64_t)phase * 0x1p-63f, &sn, &cn);
    cs[tt][p] = make_float2(cn * a.amplitude, sn * a.amplitude);
  }
  __syncthreads();

  const int qh = a.q ? a.heads : 0;
  const int per_token = (int)a.by_rows.d;
  const int c = tid % LPR, d = 8 * c;  // this lane's chunk of its row
  const bool in = d < hd;
  const float inv_hd = 1.0f / (float)hd;
  // Every lane of a wave runs the same iterations: the lanes of a row meet in shuffles.
  for (int i0 = 0; i0 < n * per_token; i0 += NR_THREADS / LPR) {
    const int i = i0 + tid / LPR;
    const bool active = i < n * per_token;
    const int tt = active ? seq_div(i, a.by_rows) : 0;
    int h = active ? i - tt * per_token : 0;
    const int64_t row = t.q0 + r0 + tt;
    const int key = key0 + tt;
    const bool is_q = h < qh, is_v = h >= qh + HK;
    if (!is_q) h -= is_v ? qh + HK : qh;
    const T* src = is_q   ? (const T*)a.q + row * a.q_st + h * a.q_sh
                   : is_v ? (const T*)a.v + row * a.v_st + h * a.v_sh
                          : (const T*)a.k + row * a.k_st + h * a.k_sh;
    float x[8];
    u32x4 raw = {0, 0, 0, 0};
    if (active && in) raw = ld128(src + d);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = unpack8<T>(raw, e);
    if (a.norm != TX_NORM_NONE) {
      float mu = 0.f;
      if (a.norm == TX_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += x[e];
        mu = nr_sum<LPR>(s) * inv_hd;
      }
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = in ? x[e] - mu : 0.f;
        s += y * y;
      }
      const float r = 1.0f / sqrtf(nr_sum<LPR>(s) * inv_hd + a.eps);
      if (!is_v) {
        const void* weight = is_q ? a.q_weight : a.k_weight;
        const void* bias = is_q ? a.q_bias : a.k_bias;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (x[e] - mu) * r;
        float w[8];
        if (weight && in) {
          nr_params<T>(weight, a.param_f32, (int64_t)h * a.param_sh + d, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= w[e];
        }
        if (bias && in) {
          nr_params<T>(bias, a.param_f32, (int64_t)h * a.param_sh + d, w);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] += w[e];
        }
      }
    }
    // The turn.
    if (a.interleaved) {
      if (!is_v) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (d + 2 * j < a.rotary) {
            const float2 w = cs[tt][(d >> 1) + j];
            const float p = x[2 * j], q = x[2 * j + 1];
            x[2 * j] = p * w.x - q * w.y;
            x[2 * j + 1] = q * w.x + p * w.y;
          }
        }
      }
    } else if (!CROSS) {
      const int hc = half >> 3;  // chunks of a half
      const bool first = c < hc, turns = c < 2 * hc && !is_v;
      const int from = (tid & 63) + (first ? hc : -hc);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __shfl(x[e], turns ? from : (tid & 63), 64);
        if (turns) {
          const float2 w = cs[tt][d - (first ? 0 : half) + e];
          x[e] = first ? x[e] * w.x - y * w.y : x[e] * w.x + y * w.y;
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
        if (at < a.rotary && !is_v) {
          const bool first = at < half;
          const float y = mine[first ? at + half : at - half];
          const float2 w = cs[tt][first ? at : at - half];
          x[e] = first ? x[e] * w.x - y * w.y : x[e] * w.x + y * w.y;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    u32x4 out = raw;
    if (!is_v)
#pragma unroll
      for (int j = 0; j < 4; ++j) out[j] = pack2<T>(x[2 * j], x[2 * j + 1]);
    if (active && in) {
      if (is_q) st128((T*)a.q_out + row * a.qo_st + h * a.qo_sh + d, out);
      else if (!is_v && a.k_out) st128((T*)a.k_out + row * a.ko_st + h * a.ko_sh + d, out);
    }
    if (!a.k_cache) continue;
    const int page = active && !is_q ? seq_page(a.s, t.b, key) : -1, slot = key & ((1 << a.s.page_log2) - 1);
    if (!a.k_scales) {
      if (page >= 0 && in)
        st128(is_v ? (T*)a.v_cache + page * a.vc_sp + h * a.vc_sh + slot * a.vc_st + d
                   : (T*)a.k_cache + page * a.kc_sp + h * a.kc_sh + slot * a.kc_st + d, out);
      continue;
    }
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, mx_magnitude<T>(x[e]));
    top = fmaxf(top, __shfl_xor(top, 1, 64));
    top = fmaxf(top, __shfl_xor(top, 2, 64));
    const int ex = mx_exponent<T>(top);
    const float inv = mx_power(-ex);
    if (page >= 0 && in) {
      uint8_t* to = is_v ? (uint8_t*)a.v_cache + page * a.vc_sp + h * a.vc_sh + slot * a.vc_st
                         : (uint8_t*)a.k_cache + page * a.kc_sp + h * a.kc_sh + slot * a.kc_st;
      st64(to + d, u32x2{mx_codes<T>(x, inv), mx_codes<T>(x + 4, inv)});
      if ((c & 3) == 0) {
        uint8_t* s = is_v ? a.v_scales + page * a.vs_sp + h * a.vs_sh + slot * a.vs_st
                          : a.k_scales + page * a.ks_sp + h * a.ks_sh + slot * a.ks_st;
        s[c >> 2] = (uint8_t)(ex + 127);
      }
    }
  }
}

template <typename T, int LPR>
static int launch_lpr(const NormRotaryArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)seq_tiles(a.s, 1, NR_TOKENS)), block(NR_THREADS);
  if (!a.interleaved && a.rotary % 16) norm_rotary_kernel<T, LPR, true><<<grid, block, 0, st>>>(a);
  else norm_rotary_kernel<T, LPR, false><<<grid, block, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
}

template <typename T>
static int launch_typed(NormRotaryArgs a, hipStream_t st) {
  a.by_rows = seq_div_by((a.q ? a.heads : 0) + (a.k_cache ? 2 : 1) * a.kv_heads);
  if (a.head_dim <= 64) return launch_lpr<T, 8>(a, st);
  if (a.head_dim <= 128) return launch_lpr<T, 16>(a, st);
  return launch_lpr<T, 32>(a, st);
}

int launch_norm_rotary_append(const NormRotaryArgs& a, int dt, hipStream_t st) {
  return dt == TX_BF16 ? launch_typed<bf16>(a, st) : launch_typed<f16>(a, st);
}

}  // namespace tx
