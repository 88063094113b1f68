// Attention over packed sequences and over a paged cache, with grouped heads.
//
//   o[t, h] = sum_j p_j v_j,   p_j = exp(s_j - max s) / sum exp(s - max s),
//   s_j = scale * q[t, h] . k[j, h / group]
#include <type_traits>

#include "attention_tiles.hpp"
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

// ------------------------------------------------------------ tiles of rows
// A workgroup of 4 waves owns 128 rows of one (sequence, K/V head), 32 per
// wave.  Row r is (token r / group, query head r % group of the K/V head), so
// that grouped heads share every K and V tile and a causal tile ends after 128
// / group tokens.  Scores are formed transposed, S^T = K Q^T on
// v_mfma_f32_32x32x16, from the key-permuted K operand, so that a lane's
// scores are, in order, the P operand of the second product; V keeps its
// natural layout and is transposed by its LDS reads (attention_tiles.hpp).
constexpr int SQ_ROWS = 128;
constexpr int SQ_THREADS = 256;
constexpr float SQ_LOG2E = 1.4426950408889634f;

typedef const __attribute__((address_space(4))) int32_t* SqConstInt;

// K and V tiles of 64 keys, global -> LDS by DMA.  One wave instruction moves
// RPI consecutive key rows, which lie in one page (page sizes are powers of
// two of at least 8): the page and the row's address are wave-uniform (scalar
// loads and arithmetic), the lane adds one constant offset.
template <typename T, int HD, bool PAGED>
struct SqLoader {
  static constexpr int CH = HD / 8;         // 16-byte chunks per row
  static constexpr int RPI = 64 / CH;       // rows per wave instruction (8 or 4)
  static constexpr int LD = AX_BN / RPI / 4;  // instructions per wave and tile (2 or 4)
  static constexpr int ELEMS = AX_BN * HD;
  const T* k;  // this K/V head's row 0 (packed) or page 0 (paged)
  const T* v;
  SqConstInt table;
  int64_t k_sp, k_st, v_sp, v_st;
  int psl, num_pages;
  int wv, last;        // last key that may be read
  int rl;              // this lane's row within an instruction's rows
  uint32_t kc, vc;     // byte offset of its chunk within a row
  uint32_t ko, vo;     // byte offset of row and chunk
  int pg[LD];          // pages of the tile that issue() loads next (looked up one tile ahead)
  int bad_from;        // first key found without a page

  __device__ __forceinline__ void init(const SeqAttnArgs& a, const SeqHead<T, PAGED>& hp, int wave, int lane) {
    k = hp.k;
    v = hp.v;
    k_st = a.k_st;
    v_st = a.v_st;
    wv = wave;
    rl = lane / CH;
    const int row = wave * RPI + rl;  // the swizzles repeat every 4 * RPI rows
    kc = 16u * (uint32_t)((lane % CH) ^ ax_kswz<HD>(row));
    vc = 16u * (uint32_t)((lane % CH) ^ ax_vswz<HD>(row));
    ko = kc + 2u * (uint32_t)rl * (uint32_t)k_st;
    vo = vc + 2u * (uint32_t)rl * (uint32_t)v_st;
    if constexpr (PAGED) {
      table = (SqConstInt)(uintptr_t)(a.s.table + (int64_t)hp.b * a.s.table_ld);
      k_sp = a.k_sp;
      v_sp = a.v_sp;
      psl = a.s.page_log2;
      num_pages = a.s.num_pages;
    }
  }
  __device__ __forceinline__ int row0(int kt, int i) const {
    return min(kt * AX_BN + (i * 4 + wv) * RPI, last & ~(RPI - 1));
  }
  __device__ __forceinline__ void lookup(int kt) {
    if constexpr (PAGED) {
#pragma unroll
      for (int i = 0; i < LD; ++i) pg[i] = table[row0(kt, i) >> psl];
    }
  }
  // Rows past the last key re-read the last one (their scores are masked).
  __device__ __forceinline__ void issue(int kt, uint32_t ks, uint32_t vs) {
    const bool full = (kt + 1) * AX_BN <= last + 1;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int r0 = row0(kt, i);
      const T* kb;
      const T* vb;
      if constexpr (PAGED) {
        int p = pg[i];
        if ((uint32_t)p >= (uint32_t)num_pages) {
          bad_from = min(bad_from, (r0 >> psl) << psl);
          p = 0;
        }
        const int slot = r0 & ((1 << psl) - 1);
        kb = k + p * k_sp + slot * k_st;
        vb = v + p * v_sp + slot * v_st;
      } else {
        kb = k + r0 * k_st;
        vb = v + r0 * v_st;
      }
      uint32_t kof = ko, vof = vo;
      if (!full) {
        const uint32_t r = (uint32_t)min(rl, last - r0);
        kof = kc + 2u * r * (uint32_t)k_st;
        vof = vc + 2u * r * (uint32_t)v_st;
      }
      const uint32_t at = (uint32_t)((i * 4 + wv) * RPI * HD * 2);
      dma16_m0(kb, kof, ks + at);
      dma16_m0(vb, vof, vs + at);
    }
  }
};

// The rows [32 wave, + 32) of a tile over the keys of the tiles [kt0, kt1):
// unnormalised o, the row sum l of its weights and the base mc (log2 units)
// they were measured from.
template <typename T, int HD, bool PAGED>
struct SqTile {
  typedef typename Mfma<T>::vec vec;
  typedef typename Mfma16<T>::vec vec16;
  typedef SqLoader<T, HD, PAGED> L;
  static constexpr int NST = HD == 128 ? 2 : 3;
  static constexpr int LDS_ELEMS = NST * 2 * L::ELEMS;
  static constexpr int LPW = 2 * L::LD;
  // fp16 weights reach 2^15 at most instead of 2^8, so that the small ones
  // stay above fp16's subnormal range for longer; bf16 has fp32's range.
  static constexpr float BIAS = std::is_same<T, f16>::value ? 7.f : 0.f;

  f32x16 o[HD / 32];
  f32x4 lsum;
  float m_run, mc;

  // q row of this lane; mylim: keys it sees; wlim_min / wlim_max: over the
  // wave's rows (wave-uniform; wlim_max 0: no rows).  Every wave of the
  // workgroup runs the same tiles.
  __device__ __forceinline__ void run(L& ld, const T* qrow, float scale, int mylim, int wlim_min, int wlim_max,
                                      int kt0, int kt1, T* lds, int lane) {
    const float NEG_INF = -__builtin_inff();
    const float c = scale * SQ_LOG2E;
    const int half = lane >> 5;
    vec qf[HD / 16];
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) qf[ks] = __builtin_bit_cast(vec, ld128(qrow + 8 * half + 16 * ks));
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) settle(qf[ks]);
    AxKOff<HD> ko;
    ko.init_perm(lane);
    AxVNatOff<HD> vn;
    vn.init(lane);
    // Row sum on the matrix cores: a 0/1 selector against P, 16 keys a step
    // (register 0 of a lane receives its own query's sum).
    vec16 sel;
    {
      const uint32_t one2 = std::is_same<T, bf16>::value ? 0x3F803F80u : 0x3C003C00u;
      const uint32_t w = (((lane >> 4) & 1) == (((lane & 15) >> 2) & 1)) ? one2 : 0u;
      sel = __builtin_bit_cast(vec16, u32x4{w, w, w, w});
    }
#pragma unroll
    for (int t = 0; t < HD / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[t][r] = 0.f;
    lsum = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run = NEG_INF;
    mc = 0.f;
    const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) T*)lds;
    auto stage = [&](int kt) { return base + (uint32_t)((kt % NST) * 2 * L::ELEMS * 2); };
    auto issue = [&](int kt) {  // tiles past the end re-read the last one
      const uint32_t s = stage(kt);
      ld.issue(min(kt, kt1 - 1), s, s + L::ELEMS * 2);
      ld.lookup(min(kt + 1, kt1 - 1));
    };
    ld.lookup(kt0);
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) issue(kt0 + s);

    for (int kt = kt0; kt < kt1; ++kt) {
      const int j0 = kt * AX_BN;
      ring_barrier<LPW * (NST - 2)>();
      issue(kt + NST - 1);
      if (j0 >= wlim_max) continue;  // no row of this wave sees these keys
      const T* Ks = lds + (kt % NST) * 2 * L::ELEMS;
      uint32_t va[HD / 32];
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) va[dt] = stage(kt) + L::ELEMS * 2 + 2u * (uint32_t)vn.off[dt];
      f32x16 s[2];
      ax_scores<T, HD>(Ks, qf, ko, s);
      if (j0 + AX_BN > wlim_min) {
        const int d = mylim - j0 - 8 * half;  // slot of key j0 + 8 half + x is seen if x < d
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[t][r] = (32 * t + ((r >> 3) << 4) + (r & 7) < d) ? s[t][r] : NEG_INF;
      }
      float mx = NEG_INF;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
      {
        const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mx),
                                                         __builtin_bit_cast(uint32_t, mx), false, false);
        mx = fmaxf(__builtin_bit_cast(float, (uint32_t)sw[0]), __builtin_bit_cast(float, (uint32_t)sw[1]));
      }
      mx *= c;
      // Re-base when a row's maximum grows past m_run + 8.
      if (__any(mx > m_run + 8.f)) {
        const float m_new = fmaxf(m_run, mx);
        const float corr = m_run == NEG_INF ? 0.f : exp2f(m_run - m_new);
#pragma unroll
        for (int j = 0; j < 4; ++j) lsum[j] *= corr;
#pragma unroll
        for (int t = 0; t < HD / 32; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[t][r] *= corr;
        m_run = m_new;
        mc = (m_run == NEG_INF ? 0.f : m_run) - BIAS;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = u >> 1, hh = u & 1;
        u32x4 vop[HD / 32];
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) {
          switch (u) {
            case 0: vop[dt] = ax_vnat_issue<HD, 0>(va[dt]); break;
            case 1: vop[dt] = ax_vnat_issue<HD, 1>(va[dt]); break;
            case 2: vop[dt] = ax_vnat_issue<HD, 2>(va[dt]); break;
            default: vop[dt] = ax_vnat_issue<HD, 3>(va[dt]); break;
          }
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][8 * hh + e], c, -mc));
        const u32x4 pk = u32x4{pack2_raw<T>(p[0], p[1]), pack2_raw<T>(p[2], p[3]), pack2_raw<T>(p[4], p[5]),
                               pack2_raw<T>(p[6], p[7])};
        const vec pf = __builtin_bit_cast(vec, pk);
        lsum = Mfma16<T>::mma(sel, __builtin_bit_cast(vec16, pk), lsum);
        ax_vnat_wait<HD / 32>(vop);
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt) o[dt] = Mfma<T>::mma32(__builtin_bit_cast(vec, vop[dt]), pf, o[dt]);
      }
    }
    ring_drain();
  }
};

// First key (of those the row needs) that has no page, over the workgroup.
__device__ __forceinline__ int sq_bad_from(int mine, int* slot, int wave, int lane) {
  if (lane == 0) slot[wave] = mine;
  __syncthreads();
  return min(min(slot[0], slot[1]), min(slot[2], slot[3]));
}

template <typename T, int HD, bool PAGED>
__global__ __launch_bounds__(SQ_THREADS, 2) void seq_attn_tile_kernel(SeqAttnArgs a, int tiles) {
  typedef SqTile<T, HD, PAGED> Tile;
  __shared__ __attribute__((aligned(16))) T lds[Tile::LDS_ELEMS];
  __shared__ int bad[4];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  // The last tiles of a sequence, which see the most keys, start first.
  const int hk = blockIdx.x % a.kv_heads;
  const SeqTile t = seq_find(a.s, a.group, SQ_ROWS, tiles - 1 - (int)(blockIdx.x / a.kv_heads));
  const int rows = t.qn * a.group, r0 = t.tile * SQ_ROWS;
  if (r0 >= rows) return;
  const int G = a.group, n = min(rows - r0, SQ_ROWS);
  const int cap = PAGED ? a.s.max_pages << a.s.page_log2 : t.kvn;
  auto keys_of = [&](int r) {  // keys that row r sees
    return max(a.causal ? t.kvn - t.qn + r / G + 1 : t.kvn, 0);
  };
  const int lim = min(keys_of(r0 + n - 1), cap);
  const int w0 = r0 + 32 * wave, wn = min(n - 32 * wave, 32);
  const int wlim_max = wn > 0 ? min(keys_of(w0 + wn - 1), cap) : 0;
  const int wlim_min = wn > 0 ? min(keys_of(w0), cap) : 0;
  const int r = min(w0 + (lane & 31), r0 + n - 1);
  const bool active = (lane & 31) < wn;
  const int64_t tok = t.q0 + r / G;
  const int h = hk * G + r - (r / G) * G;
  const int sees = keys_of(r), mylim = min(sees, cap);
  const T* qrow = (const T*)a.q + tok * a.q_st + h * a.q_sh;

  SeqHead<T, PAGED> hp;
  hp.init(a, t, hk);
  typename Tile::L ld;
  ld.init(a, hp, wave, lane);
  ld.last = lim - 1;
  ld.bad_from = cap;
  Tile tile;
  tile.lsum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) tile.o[d][e] = 0.f;
  if (lim > 0) tile.run(ld, qrow, a.scale, mylim, wlim_min, wlim_max, 0, (lim + AX_BN - 1) / AX_BN, lds, lane);
  const int bad_from = PAGED ? sq_bad_from(ld.bad_from, bad, wave, lane) : 0x7fffffff;

  const float l = tile.lsum[0];
  const bool lost = PAGED && sees > bad_from;
  // Rows without keys are 0; without a page for a key, or when every score is
  // -inf, NaN.
  const float inv = l != 0.f ? 1.0f / l : (sees > 0 ? __builtin_nanf("") : 0.f);
  float odd = 0.f;  // NaN if any value of the row is not finite
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      tile.o[d][e] = lost ? __builtin_nanf("") : tile.o[d][e] * inv;
      odd += tile.o[d][e] * 0.f;
    }
  // A value that is not finite may come from a key that the row does not see
  // (its weight of 0 times a NaN or an infinity).  Such rows run again key by
  // key; they are rare enough that nothing above pays for them.
  const uint64_t odd_lanes = __ballot(active && !lost && sees > 0 && !(odd == 0.f));
  uint32_t todo = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
  if (active && !((todo >> (lane & 31)) & 1u)) {
    T* orow = (T*)a.o + tok * a.o_st + h * a.o_sh + 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        st64(orow + 32 * d + 8 * q4, u32x2{pack2<T>(tile.o[d][4 * q4], tile.o[d][4 * q4 + 1]),
                                           pack2<T>(tile.o[d][4 * q4 + 2], tile.o[d][4 * q4 + 3])});
  }
  while (todo != 0) {
    const int i = __builtin_ctz(todo);
    todo &= todo - 1;
    const int ri = w0 + i;
    const int64_t ti = t.q0 + ri / G;
    const int hi = hk * G + ri - (ri / G) * G;
    float o[HD / 64], m, l1;
    seq_row<T, HD, PAGED>(a, hp, (const T*)a.q + ti * a.q_st + hi * a.q_sh, 0, min(keys_of(ri), cap), o, m, l1);
    T* orow = (T*)a.o + ti * a.o_st + hi * a.o_sh;
#pragma unroll
    for (int e = 0; e < HD / 64; ++e) orow[lane + 64 * e] = from_f32<T>(o[e]);
  }
}

template <typename T, int HD>
static int launch_hd(const SeqAttnArgs& a, hipStream_t st) {
  const int tiles = (int)seq_tiles(a.s, a.group, SQ_ROWS);
  const dim3 grid((unsigned)tiles * (unsigned)a.kv_heads), block(SQ_THREADS);
  if (a.paged) seq_attn_tile_kernel<T, HD, true><<<grid, block, 0, st>>>(a, tiles);
  else seq_attn_tile_kernel<T, HD, false><<<grid, block, 0, st>>>(a, tiles);
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
