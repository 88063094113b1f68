// Rotary positions and the append to a paged cache, one pass over q, k and v.
//
// Pair (x1, x2) of a head at position p turns by t = 2 pi p f.  f is kept as
// steps = f / (2 pi) in units of 2^-64 turn, so p * steps mod 2^64 is the angle
// as a fraction of a turn, exactly, however far the position: no cos / sin
// table to read or to outgrow, and no fp32 product p * f, whose error reaches
// 0.06 rad at p = 10^6.  The fraction goes to fp32 as a signed number in
// [-1/2, 1/2), relative error 2^-24.
//
// Bound by memory: 4 (heads + 2 kv_heads) head_dim bytes a token, each once.  A
// workgroup takes R tokens of one sequence; their rotary/2 angles are formed
// once, in LDS, for all heads, then every thread moves 16-byte chunks (both
// halves of a pair of chunks in the half layout, so that a turn in place never
// reads what another thread has written).
#include "seq_common.hpp"

namespace tx {

constexpr int RA_THREADS = 256;
constexpr int RA_TOKENS = 4;  // tokens a workgroup takes

// One 16-byte chunk (8 elements), or 4 interleaved pairs of it, turned by cs.
template <typename T>
__device__ __forceinline__ u32x4 ra_turn_interleaved(u32x4 x, const float2* cs) {
  u32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = unpack8<T>(x, 2 * j), b = unpack8<T>(x, 2 * j + 1);
    r[j] = pack2<T>(a * cs[j].x - b * cs[j].y, b * cs[j].x + a * cs[j].y);
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void ra_turn_half(u32x4& x1, u32x4& x2, const float2* cs) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float lo[2], hi[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float a = unpack8<T>(x1, 2 * j + e), b = unpack8<T>(x2, 2 * j + e);
      const float2 c = cs[2 * j + e];
      lo[e] = a * c.x - b * c.y;
      hi[e] = b * c.x + a * c.y;
    }
    x1[j] = pack2<T>(lo[0], lo[1]);
    x2[j] = pack2<T>(hi[0], hi[1]);
  }
}

// VEC: the rotated part splits into whole 16-byte chunks (rotary % 16 == 0 in
// the half layout, % 8 == 0 interleaved); otherwise it is turned pair by pair,
// and only what follows the next multiple of 8 moves in chunks.
template <typename T, bool VEC>
__global__ __launch_bounds__(RA_THREADS) void rotary_append_kernel(RotaryArgs a) {
  __shared__ float2 cs[RA_TOKENS][128];
  const int tid = threadIdx.x;
  const SeqTile t = seq_find(a.s, 1, RA_TOKENS, blockIdx.x);
  const int r0 = t.tile * RA_TOKENS;
  if (r0 >= t.qn) return;
  const int n = t.qn - r0 < RA_TOKENS ? t.qn - r0 : RA_TOKENS;
  const int half = a.rotary >> 1, H = a.heads, HK = a.kv_heads, hd = a.head_dim;
  const int key0 = t.kvn - t.qn + r0;  // key index of the first row

  for (int i = tid; i < n * half; i += RA_THREADS) {
    const int tt = i / half, p = i - tt * half;
    const int64_t pos = a.positions ? a.positions[t.q0 + r0 + tt] : (int64_t)(key0 + tt);
    const uint64_t phase = (uint64_t)pos * a.steps[p];
    float sn, cn;
    sincospif((float)(int64_t)phase * 0x1p-63f, &sn, &cn);
    cs[tt][p] = make_float2(cn * a.amplitude, sn * a.amplitude);
  }
  __syncthreads();

  // Units of a head of q and k: turn_units turns (a pair of chunks in the half
  // layout, a chunk interleaved, a pair of elements when not VEC), single_units
  // elements up to the next whole chunk, then chunks; of v: chunks.
  const int units = a.units, v_units = hd >> 3;
  const int qh = a.q ? H : 0;
  const int qk_units = (qh + HK) * units, per_token = (int)a.by_token.d;
  for (int i = tid; i < n * per_token; i += RA_THREADS) {
    const int tt = seq_div(i, a.by_token);
    int u = i - tt * per_token;
    const int64_t row = t.q0 + r0 + tt;
    const int key = key0 + tt;
    // Where this head's row comes from and goes to (up to two places).
    const T* src;
    T* dst0 = nullptr;
    T* dst1 = nullptr;
    const bool is_v = u >= qk_units;
    if (is_v) u -= qk_units;
    int h = seq_div(u, is_v ? a.by_v_units : a.by_units);
    u -= h * (is_v ? v_units : units);
    if (!is_v && h < qh) {
      src = (const T*)a.q + row * a.q_st + h * a.q_sh;
      dst0 = (T*)a.q_out + row * a.qo_st + h * a.qo_sh;
    } else {
      if (!is_v) h -= qh;
      src = is_v ? (const T*)a.v + row * a.v_st + h * a.v_sh : (const T*)a.k + row * a.k_st + h * a.k_sh;
      if (!is_v && a.k_out) dst0 = (T*)a.k_out + row * a.ko_st + h * a.ko_sh;
      if (a.k_cache) {
        const int page = seq_page(a.s, t.b, key), slot = key & ((1 << a.s.page_log2) - 1);
        if (page >= 0)
          dst1 = is_v ? (T*)a.v_cache + page * a.vc_sp + h * a.vc_sh + slot * a.vc_st
                      : (T*)a.k_cache + page * a.kc_sp + h * a.kc_sh + slot * a.kc_st;
      }
      if (!dst0 && !dst1) continue;
    }
    if (is_v || u >= a.turn_units + (VEC ? 0 : a.single_units)) {
      const int d = is_v ? u * 8 : a.rotary + (VEC ? 0 : a.single_units) + (u - a.turn_units - (VEC ? 0 : a.single_units)) * 8;
      const u32x4 x = ld128(src + d);
      if (dst0) st128(dst0 + d, x);
      if (dst1) st128(dst1 + d, x);
      continue;
    }
    if constexpr (VEC) {
      if (a.interleaved) {
        const u32x4 x = ra_turn_interleaved<T>(ld128(src + u * 8), &cs[tt][u * 4]);
        if (dst0) st128(dst0 + u * 8, x);
        if (dst1) st128(dst1 + u * 8, x);
      } else {
        u32x4 x1 = ld128(src + u * 8), x2 = ld128(src + half + u * 8);
        ra_turn_half<T>(x1, x2, &cs[tt][u * 8]);
        if (dst0) {
          st128(dst0 + u * 8, x1);
          st128(dst0 + half + u * 8, x2);
        }
        if (dst1) {
          st128(dst1 + u * 8, x1);
          st128(dst1 + half + u * 8, x2);
        }
      }
    } else if (u >= a.turn_units) {
      const int d = a.rotary + u - a.turn_units;
      const T x = src[d];
      if (dst0) dst0[d] = x;
      if (dst1) dst1[d] = x;
    } else {
      const int d1 = a.interleaved ? 2 * u : u, d2 = a.interleaved ? 2 * u + 1 : u + half;
      const float x1 = to_f32(src[d1]), x2 = to_f32(src[d2]);
      const float2 c = cs[tt][u];
      const T y1 = from_f32<T>(x1 * c.x - x2 * c.y), y2 = from_f32<T>(x2 * c.x + x1 * c.y);
      if (dst0) {
        dst0[d1] = y1;
        dst0[d2] = y2;
      }
      if (dst1) {
        dst1[d1] = y1;
        dst1[d2] = y2;
      }
    }
  }
}

template <typename T>
static int launch_typed(RotaryArgs a, hipStream_t st) {
  const bool vec = a.rotary % (a.interleaved ? 8 : 16) == 0;
  a.single_units = vec ? 0 : (8 - a.rotary % 8) % 8;
  a.turn_units = vec ? (a.interleaved ? a.rotary >> 3 : a.rotary >> 4) : a.rotary >> 1;
  a.units = a.turn_units + a.single_units + ((a.head_dim - a.rotary - a.single_units) >> 3);
  const int v_units = a.head_dim >> 3;
  a.by_units = seq_div_by(a.units);
  a.by_v_units = seq_div_by(v_units);
  a.by_token = seq_div_by(((a.q ? a.heads : 0) + a.kv_heads) * a.units + (a.k_cache ? a.kv_heads * v_units : 0));
  const dim3 grid((unsigned)seq_tiles(a.s, 1, RA_TOKENS)), block(RA_THREADS);
  if (vec) rotary_append_kernel<T, true><<<grid, block, 0, st>>>(a);
  else rotary_append_kernel<T, false><<<grid, block, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
}

int launch_rotary_append(const RotaryArgs& a, int dt, hipStream_t st) {
  return dt == TX_BF16 ? launch_typed<bf16>(a, st) : launch_typed<f16>(a, st);
}

}  // namespace tx
