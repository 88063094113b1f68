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
  __device__ __forceinline__ void init(const SeqAttnArgs& a, int b_, int q0, int hk) {
    k = (const T*)a.k + hk * a.k_sh + (PAGED ? 0 : (int64_t)q0 * a.k_st);
    v = (const T*)a.v + hk * a.v_sh + (PAGED ? 0 : (int64_t)q0 * a.v_st);
    b = b_;
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

// ------------------------------------------------------------ tiles of rows
// A workgroup of 4 waves owns 128 rows of one (sequence, K/V head), 32 per
// wave.  Row r is (token r / group, query head r % group of the K/V head), so
// that grouped heads share every K and V tile and a causal tile ends after 128
// / group tokens.  Scores are formed transposed, S^T = K Q^T on
// v_mfma_f32_32x32x16, from the key-permuted K operand, so that a lane's
// scores are, in order, the P operand of the second product; V keeps its
// natural layout and is transposed by its LDS reads (attention_tiles.hpp).
constexpr int SQ_ROWS = SEQ_TILE;
constexpr int SQ_THREADS = 256;
constexpr float SQ_LOG2E = 1.4426950408889634f;

// K and V tiles of 64 keys, global -> LDS by DMA.  One wave instruction moves
// RPI consecutive key rows.  Packed: one wave-uniform base a tile, a constant
// offset per lane and instruction.  Paged: an instruction's rows lie in one
// page (page sizes are powers of two of at least 8), so its base is uniform
// too; a lookup fetches the pages of 64 / LD tiles at once, one lane each, and
// turns them into byte offsets, so that an issue is two lane reads and an add
// (looked up tile by tile with scalar loads, whose wait is shared with the LDS
// reads, a chunk of 512 tokens over 32768 keys took 174 us for 151).
template <typename T, int HD, bool PAGED>
struct SqLoader {
  static constexpr int CH = HD / 8;         // 16-byte chunks per row
  static constexpr int RPI = 64 / CH;       // rows per wave instruction (8 or 4)
  static constexpr int LD = AX_BN / RPI / 4;  // instructions per wave and tile (2 or 4)
  static constexpr int ELEMS = AX_BN * HD;
  static constexpr int NOFF = PAGED ? 1 : LD;
  struct Side {
    const char* head;    // this K/V head's row 0 (packed) or page 0 (paged)
    uint32_t st;         // bytes per row
    uint32_t chunk;      // byte offset of this lane's chunk within a row
    uint32_t off[NOFF];  // of its row and chunk within a tile (paged: within an instruction's rows)
    uint32_t lo, hi;     // paged: lane x holds the offset of rows x % LD of tile base + x / LD
  };
  Side k, v;
  const int32_t* table;
  int psl, num_pages;
  uint32_t k_sp, v_sp;  // bytes per page
  int wv, last;         // last key that may be read
  int rl;               // this lane's row within an instruction's rows
  int base;
  int bad_from;         // first key found without a page (over the lane's lookups)

  __device__ __forceinline__ void init(const SeqAttnArgs& a, const SeqHead<T, PAGED>& hp, int wave, int lane) {
    wv = wave;
    rl = lane / CH;
    const int row = wave * RPI + rl;  // the swizzles repeat every 4 * RPI rows
    auto side = [&](Side& x, const T* head, int64_t st, int swz) {
      x.head = (const char*)head;
      x.st = (uint32_t)(st * 2);
      x.chunk = 16u * (uint32_t)((lane % CH) ^ swz);
#pragma unroll
      for (int i = 0; i < NOFF; ++i) x.off[i] = x.chunk + (uint32_t)(PAGED ? rl : i * 4 * RPI + row) * x.st;
    };
    side(k, hp.k, a.k_st, ax_kswz<HD>(row));
    side(v, hp.v, a.v_st, ax_vswz<HD>(row));
    if constexpr (PAGED) {
      table = a.s.table + (int64_t)hp.b * a.s.table_ld;
      base = -(1 << 30);
      psl = a.s.page_log2;
      num_pages = a.s.num_pages;
      k_sp = (uint32_t)(a.k_sp * 2);
      v_sp = (uint32_t)(a.v_sp * 2);
    }
  }
  __device__ __forceinline__ int row0(int kt, int i) const {
    return min(kt * AX_BN + (i * 4 + wv) * RPI, last & ~(RPI - 1));
  }
  __device__ __forceinline__ void lookup(int kt) {
    base = max(kt - 1, 0);  // V follows K by one tile
    const int x = threadIdx.x & 63, key = row0(base + x / LD, x % LD);
    uint32_t page = (uint32_t)table[key >> psl];
    if (page >= (uint32_t)num_pages) {  // page 0 in its place
      bad_from = min(bad_from, (key >> psl) << psl);
      page = 0;
    }
    // 32 x 32 -> 64 bits: the entry point bounds the byte strides.
    const uint32_t slot = (uint32_t)key & ((1u << psl) - 1);
    const uint64_t ko = (uint64_t)page * k_sp + slot * k.st, vo = (uint64_t)page * v_sp + slot * v.st;
    k.lo = (uint32_t)ko;
    k.hi = (uint32_t)(ko >> 32);
    v.lo = (uint32_t)vo;
    v.hi = (uint32_t)(vo >> 32);
  }
  // One tile of K or V rows to LDS byte address `to`.  Rows past the last key
  // re-read the last one (their scores are masked).
  __device__ __forceinline__ void issue(int kt, uint32_t to, const Side& x) {
    const bool full = (kt + 1) * AX_BN <= last + 1;
    to += (uint32_t)(wv * RPI * HD * 2);
    if (!PAGED && full) {
      const char* tile = x.head + (uint64_t)(uint32_t)(kt * AX_BN) * x.st;
#pragma unroll
      for (int i = 0; i < LD; ++i) dma16_m0(tile, x.off[i % NOFF], to + (uint32_t)(i * 4 * RPI * HD * 2));
      return;
    }
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int r0 = row0(kt, i);
      uint64_t at;
      if constexpr (PAGED) {
        const int at_lane = (kt - base) * LD + i;
        at = (uint32_t)__builtin_amdgcn_readlane((int)x.lo, at_lane) |
             ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)x.hi, at_lane) << 32);
      } else {
        at = (uint64_t)(uint32_t)r0 * x.st;
      }
      uint32_t o = x.off[0];
      if (!PAGED || !full) o = x.chunk + (uint32_t)min(rl, last - r0) * x.st;
      dma16_m0(x.head + at, o, to + (uint32_t)(i * 4 * RPI * HD * 2));
    }
  }
  __device__ __forceinline__ void issue_k(int kt, uint32_t to) {
    if constexpr (PAGED) {
      if (kt >= base + 64 / LD) lookup(kt);
    }
    issue(kt, to, k);
  }
  // Of the tile of issue_k's last call or the one before it (looked up by then).
  __device__ __forceinline__ void issue_v(int kt, uint32_t to) { issue(kt, to, v); }
};

// The rows [32 wave, + 32) of a tile over the keys of the tiles [kt0, kt1):
// unnormalised o, the row sum l of its weights and the base mc (log2 units)
// they were measured from.
// LEAD = 1: the scores of a tile are formed while the softmax of the one before
// it runs (its K tile is staged one tile ahead of V, two sets of scores).  At
// head dim 128, where registers allow two workgroups a CU either way: one
// prompt of 32768 tokens 3990 -> 3900 us, of 2048 48.5 -> 45 us.  At head dim 64
// its registers (181 for 128) cost workgroups: 40.4 -> 45.9 us for 16 prompts
// of up to 1021 tokens, so LEAD = 0 there.
// NST, the stages of the K and V rings: 2, for two workgroups a CU at head dim
// 128 and four at 64 (128 registers): a third stage there leaves three, 2 x 8192
// tokens 300 us for 285, 16 prompts of up to 1021 42.9 for 38.4.  (With 4 and 8
// where a call has no more workgroups than CUs, one prompt of 1024 tokens
// took 29.9 us for 25.9: what a lone workgroup waits for is not its loads.)
template <typename T, int HD, bool PAGED>
struct SqTile {
  typedef typename Mfma<T>::vec vec;
  typedef typename Mfma16<T>::vec vec16;
  typedef SqLoader<T, HD, PAGED> L;
  static constexpr int LEAD = HD == 128 ? 1 : 0;
  static constexpr int NST = 2;
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
    auto k_at = [&](int kt) { return base + (uint32_t)((kt % NST) * L::ELEMS * 2); };
    auto v_at = [&](int kt) { return base + (uint32_t)((NST + kt % NST) * L::ELEMS * 2); };
    // Tiles past the end re-read the last one.
    auto issue_k = [&](int kt) { ld.issue_k(min(kt, kt1 - 1), k_at(kt)); };
    auto issue_v = [&](int kt) { ld.issue_v(min(kt, kt1 - 1), v_at(kt)); };
    if constexpr (LEAD) issue_k(kt0);
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) {
      issue_k(kt0 + LEAD + s);
      issue_v(kt0 + s);
    }
    // Scores of one 16-wide step of the head dim, both 32-key halves.
    auto qk = [&](const T* Ks, int ks, f32x16* s) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const vec kf = *reinterpret_cast<const vec*>(Ks + 32 * t * HD + ko.off[ks]);
        s[t] = Mfma<T>::mma32(kf, qf[ks], s[t]);
      }
    };
    auto zero = [&](f32x16* s) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
    };
    // One tile: the weights and P V of tile kt from its scores sc (formed here
    // without LEAD), and with LEAD the scores sn of tile kt + 1, whose matrix
    // instructions run beside the vector work of tile kt's softmax.
    auto step = [&](int kt, f32x16* sc, f32x16* sn) {
      const int j0 = kt * AX_BN;
      ring_barrier<LPW * (NST - 2)>();  // K of tile kt + LEAD, V of tile kt
      issue_k(kt + LEAD + NST - 1);
      issue_v(kt + NST - 1);
      if (j0 >= wlim_max) return;  // no row of this wave sees these keys, nor later ones
      const T* Kn = lds + ((kt + LEAD) % NST) * L::ELEMS;
      uint32_t va[HD / 32];
#pragma unroll
      for (int dt = 0; dt < HD / 32; ++dt) va[dt] = v_at(kt) + 2u * (uint32_t)vn.off[dt];
      if constexpr (!LEAD) {
        zero(sc);
#pragma unroll
        for (int ks = 0; ks < HD / 16; ++ks) qk(Kn, ks, sc);
      }
      if (j0 + AX_BN > wlim_min) {
        const int d = mylim - j0 - 8 * half;  // slot of key j0 + 8 half + x is seen if x < d
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r) sc[t][r] = (32 * t + ((r >> 3) << 4) + (r & 7) < d) ? sc[t][r] : NEG_INF;
      }
      if constexpr (LEAD) {  // (after the last tile: scores that nothing uses)
        zero(sn);
#pragma unroll
        for (int ks = 0; ks < HD / 64; ++ks) qk(Kn, ks, sn);
      }
      // The largest score, NaN if any is (v_maximum3_f32).
      float mx = NEG_INF;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = __builtin_elementwise_maximum(mx, sc[t][r]);
      {
        const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mx),
                                                         __builtin_bit_cast(uint32_t, mx), false, false);
        mx = __builtin_elementwise_maximum(__builtin_bit_cast(float, (uint32_t)sw[0]),
                                           __builtin_bit_cast(float, (uint32_t)sw[1]));
      }
      mx *= c;
      // Re-base when a row's maximum grows past m_run + 8, or is no number.
      if (__any(!(mx <= m_run + 8.f))) {
        // A score that is NaN or +inf makes its row NaN: the row sum says so, and
        // the row sees nothing from here on (a NaN weight would make the sum of
        // the row 16 lanes away NaN too).
        const bool lost = !(mx < -NEG_INF);
        if (__any(lost)) {
          mylim = lost ? 0 : mylim;
          wlim_min = 0;
          mx = lost ? NEG_INF : mx;
#pragma unroll
          for (int j = 0; j < 4; ++j) lsum[j] = lost ? __builtin_nanf("") : lsum[j];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[t][r] = lost ? NEG_INF : sc[t][r];
        }
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
      u32x4 pk[4];
      auto weights = [&](int u) {
        const int t = u >> 1, hh = u & 1;
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][8 * hh + e], c, -mc));
        pk[u] = u32x4{pack2_raw<T>(p[0], p[1]), pack2_raw<T>(p[2], p[3]), pack2_raw<T>(p[4], p[5]),
                      pack2_raw<T>(p[6], p[7])};
      };
      if constexpr (LEAD) {
#pragma unroll
        for (int ks = HD / 64; ks < HD / 16; ++ks) qk(Kn, ks, sn);
        weights(0);
        weights(1);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
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
        if constexpr (!LEAD) weights(u);
        lsum = Mfma16<T>::mma(sel, __builtin_bit_cast(vec16, pk[u]), lsum);
        if (LEAD && u < 2) weights(u + 2);
        ax_vnat_wait<HD / 32>(vop);
#pragma unroll
        for (int dt = 0; dt < HD / 32; ++dt)
          o[dt] = Mfma<T>::mma32(__builtin_bit_cast(vec, vop[dt]), __builtin_bit_cast(vec, pk[u]), o[dt]);
      }
    };
    f32x16 sa[2];
    if constexpr (LEAD) {
      f32x16 sb[2];
      ring_barrier<LPW * (NST - 1)>();  // K of the first tile
      zero(sa);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks) qk(lds + (kt0 % NST) * L::ELEMS, ks, sa);
      for (int kt = kt0; kt < kt1; kt += 2) {
        step(kt, sa, sb);
        if (kt + 1 < kt1) step(kt + 1, sb, sa);
      }
    } else {
      for (int kt = kt0; kt < kt1; ++kt) step(kt, sa, sa);
    }
    ring_drain();
  }
};

// First key (of those the row needs) that has no page, over the workgroup.
__device__ __forceinline__ int sq_bad_from(int mine, int* slot, int wave, int lane) {
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) mine = min(mine, __shfl_xor(mine, x, 64));
  if (lane == 0) slot[wave] = mine;
  __syncthreads();
  return min(min(slot[0], slot[1]), min(slot[2], slot[3]));
}

// The kernel's first argument, read where this is called and not before.
__device__ __forceinline__ const SeqAttnArgs& sq_args_again() {
  uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const SeqAttnArgs*)(const __attribute__((address_space(4))) SeqAttnArgs*)p;
}

// Rows whose result is not finite though the sum of their weights is, up to 16
// by one wave (lane: row lane & 15, r of the sequence's; `need`), after they are
// stored.  What a row must come to:
// sum_j w_j v_j over the keys it sees, w_j its fp32 weight, in IEEE arithmetic.
// The first pass also adds 0 x v of the keys that the mask hides (NaN where v
// is not finite), and its unnormalised sums pass fp32's range where values near
// the end of it are added up.  So:
//  * Look through the keys for values that are not finite.  Of 32 keys with
//    any, note per element which infinities the row sees (a NaN counts as
//    both): MFMAs of 0/1 operands, (weight > 0) x (value is that infinity).
//    This ends where it explains every infinity and NaN that is stored, at the
//    first bad key as a rule: they are right then.
//  * Rows with something unexplained run again with normalised weights over
//    values whose infinities and NaN are replaced by 0, the noted ones added.
// 4096 causal tokens, 8 / 2 heads of 64, an infinity in v of the first token: 67
// us for 61 of a clean call, of the last one 570 (one row after another, key by
// key: 15 and 16 ms).
// Loads go straight to registers: no other wave need take part.  16 rows, and
// the call's arguments read again here, so that the kernels around this keep
// their registers (32 rows and arguments held across put 58 to 90 of them in
// scratch memory: 32 short streams took 32 us for 21).
// po: not nullptr: the row's partial result.
template <typename T, int HD, bool PAGED>
__device__ __forceinline__ void sq_odd_rows(int b, int q0, int hk, int r, bool need, int sees, int j0, float m, float l,
                                            float bias, float* po, int lane) {
  typedef typename Mfma16<T>::vec vec;
  constexpr uint32_t EXP = std::is_same<T, bf16>::value ? 0x7F80u : 0x7C00u;  // all ones: not finite
  constexpr uint32_t ONE = std::is_same<T, bf16>::value ? 0x3F80u : 0x3C00u;
  const float INF = __builtin_inff();
  const SeqAttnArgs& a = sq_args_again();
  SeqHead<T, PAGED> hp;
  hp.init(a, b, q0, hk);
  const int col = lane & 15, g = lane >> 4;
  const int i0 = seq_div(r, a.by_group);
  const int64_t tok = q0 + i0;
  const int h = hk * a.group + r - i0 * a.group;
  const T* qrow = (const T*)a.q + tok * a.q_st + h * a.q_sh + 8 * g;
  T* orow = (T*)a.o + tok * a.o_st + h * a.o_sh + 4 * g;
  const float c = a.scale * SQ_LOG2E, mc = (m == -INF ? 0.f : m) - bias;
  sees = need ? sees : 0;
  int lim = sees;
#pragma unroll
  for (int x = 8; x > 0; x >>= 1) lim = max(lim, __shfl_xor(lim, x, 64));
  lim = seq_uni(lim);

  // Weights of the 32 keys from k0 on: w[x][e] is of key k0 + 16 x + 4 g + e, 0
  // where masked.
  auto key_of = [&](int k0, int x, int e) { return k0 + 16 * x + 4 * g + e; };
  auto weights = [&](int k0, f32x4* w) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const T *kr, *vr, *qr = qrow;
      hp.at(a, min(k0 + 16 * x + col, lim - 1), kr, vr);
      asm volatile("" : "+v"(qr), "+v"(kr));
      w[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
        w[x] = Mfma16<T>::mma(__builtin_bit_cast(vec, ld128(kr + 32 * i + 8 * g)),
                              __builtin_bit_cast(vec, ld128(qr + 32 * i)), w[x]);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[x][e] = key_of(k0, x, e) < sees ? exp2f(__builtin_fmaf(w[x][e], c, -mc)) : 0.f;
    }
  };
  // Element 16 d + col of the values of the keys that w's weights are of.
  auto values = [&](int k0, int d, uint32_t* v) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const T *kr, *vr;
      const int j = min(k0 + 16 * x + 4 * g, (lim - 1) & ~3);  // four keys lie in one page
      int left = lim - 1 - j;
      hp.at(a, j, kr, vr);
      vr += col + 16 * d;
      asm volatile("" : "+v"(vr), "+v"(left));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[4 * x + e] = __builtin_bit_cast(uint16_t, vr[(uint64_t)(uint32_t)min(e, left) * (uint32_t)a.v_st]);
    }
  };

  // Bit 4 d + e: element 16 d + 4 g + e of the row.  What is +inf or NaN, what
  // -inf or NaN, and the infinities seen that explain it.
  uint32_t odd_p = 0, odd_n = 0, pos = 0, neg = 0;
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) {
    float y[4];
    if (po) load4<float>(po + 16 * d + 4 * g, y);
    else load4<T>(orow + 16 * d, y);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      odd_p |= (need && !(y[e] < INF) ? 1u : 0u) << (4 * d + e);
      odd_n |= (need && !(y[e] > -INF) ? 1u : 0u) << (4 * d + e);
    }
  }
  bool bad = false;
#pragma unroll 1
  for (int k0 = j0; k0 < lim; k0 += 32) {
    if ((k0 - j0) % 64 == 0) {  // look through 64 keys
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < HD / 8; ++i) {
        const T *kr, *vr;
        const int x = 64 * i + lane;
        hp.at(a, min(k0 + x / (HD / 8), lim - 1), kr, vr);
        const u32x4 y = ld128(vr + x % (HD / 8) * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          any |= (y[e] & EXP) == EXP || (y[e] & (EXP << 16)) == EXP << 16 ? 1u : 0u;
      }
      bad = __any(any != 0);
      if (!bad) k0 += 32;
    }
    if (!bad) continue;
    f32x4 w[2];
    weights(k0, w);
    // 0/1 operands: seen with a weight, seen with a weight of 0 (which is NaN
    // times an infinity).
    u32x4 some, zero;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t s = w[e >> 2][e & 3] > 0.f ? ONE : 0;
      const uint32_t z = !s && key_of(k0, e >> 2, e & 3) < sees ? ONE : 0;
      some[e >> 1] = e & 1 ? some[e >> 1] | s << 16 : s;
      zero[e >> 1] = e & 1 ? zero[e >> 1] | z << 16 : z;
    }
#pragma unroll 1
    for (int d = 0; d < HD / 16; ++d) {
      uint32_t v[8];
      values(k0, d, v);
      u32x4 vp, vn, vz;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t xp = v[e] == EXP || (v[e] & 0x7FFFu) > EXP ? ONE : 0;
        const uint32_t xn = v[e] == (EXP | 0x8000u) || (v[e] & 0x7FFFu) > EXP ? ONE : 0;
        vp[e >> 1] = e & 1 ? vp[e >> 1] | xp << 16 : xp;
        vn[e >> 1] = e & 1 ? vn[e >> 1] | xn << 16 : xn;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) vz[e] = vp[e] | vn[e];
      const f32x4 none = {0.f, 0.f, 0.f, 0.f};
      const f32x4 tz = Mfma16<T>::mma(__builtin_bit_cast(vec, vz), __builtin_bit_cast(vec, zero), none);
      const f32x4 tp = Mfma16<T>::mma(__builtin_bit_cast(vec, vp), __builtin_bit_cast(vec, some), tz);
      const f32x4 tn = Mfma16<T>::mma(__builtin_bit_cast(vec, vn), __builtin_bit_cast(vec, some), tz);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        pos |= (tp[e] > 0.f ? 1u : 0u) << (4 * d + e);
        neg |= (tn[e] > 0.f ? 1u : 0u) << (4 * d + e);
      }
    }
    if (__all(!(odd_p & ~pos) && !(odd_n & ~neg))) return;
  }
  bool again = (odd_p & ~pos) || (odd_n & ~neg);
  again = __shfl_xor((int)again, 16, 64) || again;
  again = __shfl_xor((int)again, 32, 64) || again;
  // fp16 weights stay above its subnormal range.
  constexpr float UP = std::is_same<T, f16>::value ? 0x1p15f : 1.f;
  const float f = (l != 0.f ? 1.0f / l : 0.f) * UP;
  f32x4 o[HD / 16];
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int k0 = j0; k0 < lim; k0 += 32) {
    uint32_t v[HD / 16][8];  // asked for before the keys, whose loads they overlap
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) values(k0, d, v[d]);
    f32x4 w[2];
    weights(k0, w);
    const u32x4 pw = {pack2<T>(w[0][0] * f, w[0][1] * f), pack2<T>(w[0][2] * f, w[0][3] * f),
                      pack2<T>(w[1][0] * f, w[1][1] * f), pack2<T>(w[1][2] * f, w[1][3] * f)};
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) {
      u32x4 vv;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t x = (v[d][e] & EXP) == EXP ? 0 : v[d][e];
        vv[e >> 1] = e & 1 ? vv[e >> 1] | x << 16 : x;
      }
      o[d] = Mfma16<T>::mma(__builtin_bit_cast(vec, vv), __builtin_bit_cast(vec, pw), o[d]);
    }
  }
  if (!again) return;
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) {
    float y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int at = 4 * d + e;
      y[e] = o[d][e] * (1.f / UP) + ((pos >> at) & 1 ? INF : 0.f) + ((neg >> at) & 1 ? -INF : 0.f);
    }
    if (po) store4<float>(po + 16 * d + 4 * g, y);
    else store4<T>(orow + 16 * d, y);
  }
}

// Rows [r0, r0 + 128) of a sequence over the keys [j0, j1) (j0 and, but for
// the last part, j1 multiples of 64).  part, ml: where the partial results of
// the tile's rows go, or nullptr for the output.
template <typename T, int HD, bool PAGED>
__device__ __forceinline__ void sq_tile_item(const SeqAttnArgs& a, int b, int q0, int qn, int kvn, int hk, int r0,
                                             int j0, int j1, float* part, float* ml, T* lds, int* bad, int lane, int wave) {
  typedef SqTile<T, HD, PAGED> Tile;
  const int G = a.group, n = min(qn * G - r0, SQ_ROWS);
  const int cap = PAGED ? a.s.max_pages << a.s.page_log2 : kvn;
  auto keys_of = [&](int r) {  // keys that row r sees
    return max(a.causal ? kvn - qn + seq_div(r, a.by_group) + 1 : kvn, 0);
  };
  const int lim = seq_uni(min(min(keys_of(r0 + n - 1), cap), j1));
  const int w0 = r0 + 32 * wave, wn = min(n - 32 * wave, 32);
  const int wlim_max = seq_uni(wn > 0 ? min(keys_of(w0 + wn - 1), lim) : 0);
  const int wlim_min = seq_uni(wn > 0 ? min(keys_of(w0), lim) : 0);
  const int r = min(w0 + (lane & 31), r0 + n - 1);
  const bool active = (lane & 31) < wn;
  const int i0 = seq_div(r, a.by_group);
  const int64_t tok = q0 + i0;
  const int h = hk * G + r - i0 * G;
  const int sees = keys_of(r);

  SeqHead<T, PAGED> hp;
  hp.init(a, b, q0, hk);
  typename Tile::L ld;
  ld.init(a, hp, wave, lane);
  ld.last = lim - 1;
  ld.bad_from = cap;
  Tile tile;
  tile.lsum = f32x4{0.f, 0.f, 0.f, 0.f};
  tile.m_run = -__builtin_inff();
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) tile.o[d][e] = 0.f;
  if (lim > j0)
    tile.run(ld, (const T*)a.q + tok * a.q_st + h * a.q_sh, a.scale, min(sees, cap), wlim_min, wlim_max, j0 / AX_BN,
             (lim + AX_BN - 1) / AX_BN, lds, lane);
  const int bad_from = PAGED ? sq_bad_from(ld.bad_from, bad, wave, lane) : 0x7fffffff;

  // Rows without keys are 0; without a page for a key, or when every score is
  // -inf, NaN.  (Of a part, l = 0 says nothing yet: the join decides.)
  const float l = tile.lsum[0];
  const bool lost = PAGED && sees > bad_from && bad_from < j1;
  const float none = part || sees <= 0 ? 0.f : __builtin_nanf("");
  const float inv = lost ? __builtin_nanf("") : (l != 0.f ? 1.0f / l : none);
  if (PAGED && __any(sees <= 0)) {  // (0 weights times a value that is not finite are not 0)
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e) tile.o[d][e] = sees > 0 ? tile.o[d][e] : 0.f;
  }
  float odd = 0.f;  // NaN if any value of the row is not finite
#pragma unroll
  for (int d = 0; d < HD / 32; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) odd += tile.o[d][e] * 0.f;
  const float by = sees > 0 ? inv : 0.f;
  if (active && !part) {
    T* orow = (T*)a.o + tok * a.o_st + h * a.o_sh + 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        st64(orow + 32 * d + 8 * q4, u32x2{pack2<T>(tile.o[d][4 * q4] * by, tile.o[d][4 * q4 + 1] * by),
                                           pack2<T>(tile.o[d][4 * q4 + 2] * by, tile.o[d][4 * q4 + 3] * by)});
  } else if (active) {
    float* po = part + (r - r0) * HD;
#pragma unroll
    for (int d = 0; d < HD / 32; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        *reinterpret_cast<f32x4*>(po + 32 * d + 8 * q4 + 4 * (lane >> 5)) =
            f32x4{tile.o[d][4 * q4] * by, tile.o[d][4 * q4 + 1] * by, tile.o[d][4 * q4 + 2] * by, tile.o[d][4 * q4 + 3] * by};
    if (lane < 32) {  // (a sum that is no number: the row is NaN)
      ml[2 * (r - r0)] = lost || !(l == l) ? __builtin_nanf("") : tile.m_run;
      ml[2 * (r - r0) + 1] = l * exp2f(-Tile::BIAS);
    }
  }
  // (l = 0: every score is -inf; of a part, hidden keys are no reason for NaN)
  const uint64_t odd_lanes = __ballot(active && !lost && sees > j0 && l == l && (l != 0.f || part) && !(odd == 0.f));
  const uint32_t odd_rows = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
  if (__builtin_expect(odd_rows == 0, 1)) return;
#pragma unroll 1
  for (int x = 0; x < 32; x += 16) {
    if (!(odd_rows & (0xFFFFu << x))) continue;
    const int row = x + (lane & 15), ri = min(w0 + row, r0 + n - 1);
    sq_odd_rows<T, HD, PAGED>(b, q0, hk, ri, (odd_rows >> row) & 1u, min(keys_of(ri), lim), j0, __shfl(tile.m_run, row, 64),
                              __shfl(l, row, 64), Tile::BIAS, part ? part + (ri - r0) * HD : nullptr, lane);
  }
}

// ------------------------------------------------------------- packed prompts
template <typename T, int HD>
__global__ __launch_bounds__(SQ_THREADS, HD == 64 ? 4 : 2) void seq_attn_packed_kernel(SeqAttnArgs a, SeqOrder order) {
  __shared__ __attribute__((aligned(16))) T lds[SqTile<T, HD, false>::LDS_ELEMS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  int hk;
  const SeqTile t = seq_ordered(a.s, a.group, SQ_ROWS, order, a.kv_heads, (int)blockIdx.x, hk);
  const int r0 = t.tile * SQ_ROWS;
  if (r0 >= t.qn * a.group) return;
  sq_tile_item<T, HD, false>(a, t.b, t.q0, t.qn, t.qn, hk, r0, 0, 0x7fffffff, nullptr, nullptr, lds, nullptr, lane, wave);
}

// -------------------------------------------------------------- few rows
// Up to 16 rows (one token's query heads of a K/V head, or a few tokens')
// against one part of the keys: bound by reading K and V once.  Each of the 4
// waves takes blocks of 32 keys by itself, no barrier between them.  Its K and
// V rows come by DMA, whole rows a wave instruction (loads in the order of the
// MFMA operand, 16 rows x 64 bytes, reach 5.9 TB/s where whole rows reach 6.8),
// into the wave's own LDS; K is read as the A operand of S^T = K Q^T (16 keys
// x 32 dims), V transposed as that of o^T += V^T P^T.  K's rows are replaced by
// the next block's once its scores are formed, V's once it is used, in each of
// the 8 waves of a CU (16 at head dim 64).  K's transfer lies beside V's and the
// softmax; V's does not reach into the scores: the wait for q that the compiler
// places before the first of them counts the page lookup behind the DMAs, but
// not the DMAs, and so drains them.  S^T leaves lane l the keys 4 (l >> 4)
// .. + 3 of both 16-key halves of row l & 15, which is a P operand as it stands
// if V's rows are taken in that order.  The waves' results meet in LDS at the
// end.
template <typename T, int HD>
struct SqFew {
  typedef typename Mfma16<T>::vec vec;
  static constexpr int CH = HD / 8, RPI = 64 / CH, LDB = 32 / RPI;  // rows per instruction, instructions per block
  static constexpr int ELEMS = 32 * HD;                             // a block of K or V; o of 16 rows in fp32
  static constexpr int WAVE_ELEMS = 2 * ELEMS;
  static constexpr float BIAS = SqTile<T, HD, true>::BIAS;
  // Instruction x moves the keys LDB (lane / CH) + x, so that a lane's keys lie
  // in one page (LDB divides 8); they land at LDS row x RPI + lane / CH.  The
  // 16-byte chunks of a key are xor-ed for the reads: 16 keys at one chunk (K),
  // 8 keys x 32 bytes (V) fall on different banks.
  static __device__ __forceinline__ int lds_row(int key) { return key % LDB * RPI + key / LDB; }
  static __device__ __forceinline__ int kswz(int key) {
    return HD == 128 ? key & 15 : (key & 3) | ((key >> 1) & 4);
  }
  static __device__ __forceinline__ int vswz(int key) { return HD == 128 ? (key & 7) << 1 : (key & 3) << 1; }
};

template <typename T, int HD>
__device__ __forceinline__ void sq_few_item(const SeqAttnArgs& a, const SeqWork& w, int hk, int r0, int j0, int j1,
                                            float* part, float* ml, T* lds, float* stat, int* bad, int lane,
                                            int wave) {
  typedef SqFew<T, HD> F;
  typedef typename F::vec vec;
  const float NEG_INF = -__builtin_inff();
  const float c = a.scale * SQ_LOG2E;
  const int G = a.group, n = min(w.qn * G - r0, w.cut.tile_rows);
  const int cap = a.s.max_pages << a.s.page_log2, ps1 = (1 << a.s.page_log2) - 1;
  auto keys_of = [&](int r) { return max(a.causal ? w.kvn - w.qn + seq_div(r, a.by_group) + 1 : w.kvn, 0); };
  const int lim = seq_uni(min(min(keys_of(r0 + n - 1), cap), j1));
  const int col = lane & 15, g = lane >> 4;
  const int r = r0 + min(col, n - 1);
  const int i0 = seq_div(r, a.by_group);
  const int64_t tok = w.q0 + i0;
  const int h = hk * G + r - i0 * G;
  const int mylim = min(keys_of(r), lim);
  SeqHead<T, true> hp;
  hp.init(a, w.b, w.q0, hk);
  const int32_t* table = a.s.table + (int64_t)w.b * a.s.table_ld;

  vec qf[HD / 32];
  {
    const T* qrow = (const T*)a.q + tok * a.q_st + h * a.q_sh + 8 * g;
#pragma unroll
    for (int ks = 0; ks < HD / 32; ++ks) qf[ks] = __builtin_bit_cast(vec, ld128(qrow + 32 * ks));
  }
  vec ones;
  {
    const uint32_t one2 = std::is_same<T, bf16>::value ? 0x3F803F80u : 0x3C003C00u;
    ones = __builtin_bit_cast(vec, u32x4{one2, one2, one2, one2});
  }
  f32x4 o[HD / 16], lsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = NEG_INF, mc = 0.f;
  int bad_from = cap;

  // A lane's keys of a block.  Keys past the last re-read the last.  Page and
  // slot parts of an address are 32 x 32 -> 64 bit products (the entry point
  // bounds the strides).
  auto key0 = [&](int kb) { return min(kb + lane / F::CH * F::LDB, (lim - 1) & ~(F::LDB - 1)); };
  auto lookup = [&](int kb) { return (uint32_t)table[key0(kb) >> a.s.page_log2]; };
  T* ks = lds + wave * F::WAVE_ELEMS;
  T* vs = ks + F::ELEMS;
  auto load = [&](int kb, uint32_t page, T* to, const T* head, int64_t sp, int64_t st, auto swz) {
    const int key = key0(kb), left = lim - 1 - key;
    if (page >= (uint32_t)a.s.num_pages) {  // page 0 in the place of one that is not there
      bad_from = min(bad_from, key & ~ps1);
      page = 0;
    }
    const uint32_t row_bytes = (uint32_t)(st * 2);
    const char* row = (const char*)head + (uint64_t)page * (uint32_t)(sp * 2) + (uint32_t)(key & ps1) * row_bytes;
#pragma unroll
    for (int x = 0; x < F::LDB; ++x)
      dma16_once(row + (uint32_t)min(x, left) * row_bytes + 16u * ((lane % F::CH) ^ swz(lane / F::CH * F::LDB + x)),
                 to + x * F::RPI * HD);
  };
  auto load_k = [&](int kb, uint32_t page) { load(kb, page, ks, hp.k, a.k_sp, a.k_st, F::kswz); };
  auto load_v = [&](int kb, uint32_t page) { load(kb, page, vs, hp.v, a.v_sp, a.v_st, F::vswz); };
  const uint32_t vbase = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) T*)vs;
  // Transposing reads: lane j of a 16-lane group g addresses key 4 g + j / 4
  // (and + 16) at dims 16 d + 4 (j % 4) and receives dim 16 d + j of 4 keys.
  const int vkey = 4 * g + (col >> 2);
  const uint32_t vrow = vbase + (uint32_t)(F::lds_row(vkey) * HD * 2 + (col & 1) * 8);
  const int vx = (col & 3) >> 1, vsw = F::vswz(vkey);
  const T* krow = ks + F::lds_row(col) * HD;
  const int ksw = F::kswz(col);
  auto compute = [&](int kb, uint32_t page, bool more) {
    // This block's K rows are there: only its V rows may still be on the way
    // (a page lookup among them makes the wait stricter).
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(F::LDB) : "memory");
    float s[8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < HD / 32; ++i)
        acc = Mfma16<T>::mma(__builtin_bit_cast(vec, ld128(krow + 16 / F::LDB * x * HD + (((4 * i + g) ^ ksw) << 3))), qf[i], acc);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[4 * x + e] = (kb + 16 * x + 4 * g + e < mylim) ? acc[e] : NEG_INF;
    }
    if (more) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read
      load_k(kb + 128, page);
    }
    float mx = NEG_INF;
#pragma unroll
    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, s[e]);
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    mx *= c;
    if (__any(mx > m_run + 8.f)) {
      const float m_new = fmaxf(m_run, mx);
      const float corr = m_run == NEG_INF ? 0.f : exp2f(m_run - m_new);
      lsum *= corr;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[d] *= corr;
      m_run = m_new;
      mc = (m_run == NEG_INF ? 0.f : m_run) - F::BIAS;
    }
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], c, -mc));
    const vec pf = __builtin_bit_cast(vec, u32x4{pack2_raw<T>(p[0], p[1]), pack2_raw<T>(p[2], p[3]),
                                                 pack2_raw<T>(p[4], p[5]), pack2_raw<T>(p[6], p[7])});
    lsum = Mfma16<T>::mma(ones, pf, lsum);
    // This block's V rows: only the next one's K may still be on the way.
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(F::LDB) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int d4 = 0; d4 < HD / 64; ++d4) {
      u32x4 vop[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t at = vrow + (uint32_t)((((2 * (4 * d4 + i)) ^ vsw) + vx) << 4);
        u32x2 lo, hi;
        asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(lo) : "v"(at));
        asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi) : "v"(at), "n"(16 / F::LDB * HD * 2));
        vop[i] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
      ax_vnat_wait<4>(vop);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[4 * d4 + i] = Mfma16<T>::mma(__builtin_bit_cast(vec, vop[i]), pf, o[4 * d4 + i]);
    }
    if (more) load_v(kb + 128, page);  // (every read above has been waited for)
  };

  const int first = j0 + 32 * wave;
  if (first < lim) {
    uint32_t page = lookup(first), next = lookup(first + 128);
    load_k(first, page);
    load_v(first, page);
    for (int kb = first; kb < lim; kb += 128) {
      page = next;
      next = lookup(kb + 256);
      compute(kb, page, kb + 128 < lim);
    }
  }

  // Join the waves: o in fp32 over each wave's K block, m and l beside it.
  if (threadIdx.x == 0) *bad = cap;
  float* ow = (float*)ks;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  float* sm = stat + wave * 16;
  float* sl = stat + 64 + wave * 16;
  int* sagain = (int*)(stat + 128);
  __syncthreads();
  if (bad_from < cap) atomicMin(bad, bad_from);
#pragma unroll
  // (4-value chunks xor the row: 16 rows at one chunk would share 4 banks)
  for (int d = 0; d < HD / 16; ++d) *reinterpret_cast<f32x4*>(ow + col * HD + 4 * ((4 * d + g) ^ col)) = o[d];
  if (g == 0) {
    sm[col] = m_run;
    sl[col] = lsum[0];
  }
  if (threadIdx.x < 16) sagain[threadIdx.x] = 0;
  __syncthreads();
  const int lost_from = *bad;
  constexpr int DT = HD / 16;  // dims a thread joins: 16 threads a row
  const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 4;
  const float* s0 = stat + row;
  float M = fmaxf(fmaxf(s0[0], s0[16]), fmaxf(s0[32], s0[48]));
  const float M0 = M == NEG_INF ? 0.f : M;
  float wt[4], L = 0.f;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    wt[x] = exp2f(s0[16 * x] - M0);
    L += wt[x] * s0[64 + 16 * x];
  }
  const int rr = r0 + min(row, n - 1);
  const int sees = keys_of(rr);
  const bool active = row < n, lost = sees > lost_from && lost_from < j1;
  const float none = part || sees <= 0 ? 0.f : __builtin_nanf("");
  const float inv = L != 0.f ? 1.0f / L : none;
  float res[DT], odd = 0.f;
#pragma unroll
  for (int y = 0; y < DT / 4; ++y) {
    f32x4 ov[4];  // a wave without keys for the row left 0 here, its weight is 0 too
#pragma unroll
    for (int x = 0; x < 4; ++x) ov[x] = *reinterpret_cast<const f32x4*>((const float*)(lds + x * F::WAVE_ELEMS) + row * HD + 64 * y + (d0 ^ 4 * row));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float v = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v = __builtin_fmaf(wt[x], ov[x][e], v);
      }
      v = lost ? __builtin_nanf("") : (sees > 0 ? v * inv : 0.f);  // (0 times what is not finite is not 0)
      res[4 * y + e] = v;
      odd += v * 0.f;
    }
  }
  // (as in a tile)
  const bool redo = active && !lost && sees > j0 && L == L && (L != 0.f || part) && !(odd == 0.f);
  if (redo) sagain[row] = 1;
  __syncthreads();
  const int ir = seq_div(rr, a.by_group);
  const int64_t tk = w.q0 + ir;
  const int hh = hk * G + rr - ir * G;
  if (active) {
    if (part) {
      float* po = part + row * HD + d0;
#pragma unroll
      for (int y = 0; y < DT / 4; ++y) store4<float>(po + 64 * y, res + 4 * y);
      if ((threadIdx.x & 15) == 0) {  // (a sum that is no number: the row is NaN)
        ml[2 * row] = lost || !(L == L) ? __builtin_nanf("") : M;
        ml[2 * row + 1] = L * exp2f(-F::BIAS);
      }
    } else {
      T* orow = (T*)a.o + tk * a.o_st + hh * a.o_sh + d0;
#pragma unroll
      for (int y = 0; y < DT / 4; ++y) store4<T>(orow + 64 * y, res + 4 * y);
    }
  }
  if (__builtin_expect(!__any(sagain[col]), 1)) return;  // (the same in every wave)
  // Wave 0 sees to the rows that are not finite, once all are stored.
  if ((threadIdx.x & 15) == 0) {
    stat[row] = M;
    stat[64 + row] = L;
  }
  __syncthreads();
  if (wave != 0) return;
  const int ro = min(col, n - 1);
  sq_odd_rows<T, HD, true>(w.b, w.q0, hk, r0 + ro, col < n && sagain[col] != 0, min(keys_of(r0 + ro), lim), j0, stat[col],
                           stat[64 + col], F::BIAS, part ? part + ro * HD : nullptr, lane);
}

// ---------------------------------------------------------------- paged calls
__host__ __device__ inline SeqShape sq_shape(const SeqAttnArgs& a) {
  return SeqShape{a.group, a.kv_heads, a.cus, a.head_dim == 128 ? 2 : 1, a.few_parts, a.few};
}

// Persistent workgroups over the items of a call (SeqWalk); a grid of at most
// the items, so every workgroup's loop ends.
template <typename T, int HD, bool FEW_ONLY>
__global__ __launch_bounds__(SQ_THREADS, HD == 64 ? (FEW_ONLY ? 4 : 3) : 2) void seq_attn_paged_kernel(SeqAttnArgs a) {
  constexpr int TILE_ELEMS = SqTile<T, HD, true>::LDS_ELEMS, FEW_ELEMS = 4 * SqFew<T, HD>::WAVE_ELEMS;
  constexpr int ELEMS = FEW_ONLY || FEW_ELEMS > TILE_ELEMS ? FEW_ELEMS : TILE_ELEMS;
  __shared__ __attribute__((aligned(16))) T lds[ELEMS];
  __shared__ float stat[144];
  __shared__ int bad[4];
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const SeqShape sh = sq_shape(a);
  __shared__ int seqs[SeqWalk::LDS_INTS];
  SeqWalk walk;
  walk.init(a.s, sh, false, seqs);
  SeqWork w;
  for (int i = blockIdx.x; walk.find(a.s, sh, false, i, w); i += gridDim.x) {
    // An item's lane constants are formed within it: held across the items
    // they cost the registers that its loads need (56 spills).
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    // Item u of a sequence: its (part, K/V head) pairs first, then its tiles:
    // the tiles that share keys meet on one XCD when the pairs are a multiple
    // of 8.
    const int u = i - w.item, np = w.cut.parts * a.kv_heads;
    const int tile = w.cut.tiles > 1 ? seq_uni(u / np) : 0, pair = u - tile * np;
    const int p = seq_uni(seq_div(pair, a.by_kv_heads)), hk = pair - p * a.kv_heads;
    const int j0 = p * w.cut.part_keys, j1 = p + 1 < w.cut.parts ? j0 + w.cut.part_keys : 0x7fffffff;
    // Partial results of a sequence: by tile, part, K/V head, row of the tile.
    const int r0 = tile * w.cut.tile_rows;
    float *part = nullptr, *ml = nullptr;
    if (w.cut.parts > 1) {
      const int64_t at = w.partial + r0 * np + pair * min(w.qn * a.group - r0, w.cut.tile_rows);
      part = a.ws + at * HD;
      ml = a.ws_ml + at * 2;
    }
    if constexpr (FEW_ONLY) {
      sq_few_item<T, HD>(a, w, hk, r0, j0, j1, part, ml, lds, stat, bad, lane, wave);
    } else {
      if (w.cut.few) sq_few_item<T, HD>(a, w, hk, r0, j0, j1, part, ml, lds, stat, bad, lane, wave);
      else sq_tile_item<T, HD, true>(a, w.b, w.q0, w.qn, w.kvn, hk, r0, j0, j1, part, ml, lds, bad, lane, wave);
    }
    __syncthreads();  // LDS belongs to the next item
  }
}

// Joins the parts of each row: o = sum_p w_p o_p / sum_p w_p, w_p = l_p 2^(m_p
// - max m), parts in one order whatever runs first.  Rows of at most
// SEQ_WAVE_PARTS parts take a wave each, others a workgroup each.  Its time is
// a chain of loads (sequence, then m and l beside o), so the o of the first
// parts is asked for before their weights are known.
template <typename T, int HD, bool WAVE>
__device__ __forceinline__ void sq_join_row(const SeqAttnArgs& a, const SeqWork& w, int hk, int r, int tid,
                                            float (*red)[4]) {
  constexpr int LPR = HD / 4;                    // lanes of 4 dims a part
  constexpr int GRP = (WAVE ? 64 : 256) / LPR;   // parts at a time
  constexpr int NP = WAVE ? SEQ_WAVE_PARTS / GRP : 8;  // o values asked for at once
  constexpr int MLS = WAVE ? 1 : 4;              // parts whose m and l a lane holds
  static_assert((WAVE ? SEQ_WAVE_PARTS : SEQ_JOIN_PARTS) <= 64 * MLS, "a row's parts are held one a lane");
  const int lane = tid & 63;
  if (WAVE) tid = lane;
  const float NEG_INF = -__builtin_inff();
  const int tr = w.cut.tile_rows;
  const int tile = w.cut.tiles == 1 ? 0 : (w.cut.few ? seq_uni(r / tr) : r / SQ_ROWS), r0 = tile * tr;
  const int n = min(w.qn * a.group - r0, tr);
  const int64_t at = w.partial + r0 * w.cut.parts * a.kv_heads + hk * n + r - r0;  // of part 0
  // Byte offsets from there to a part's: at most (2 CUs + kv_heads) times a
  // tile's rows, below 2^32.
  const char *first = (const char*)(a.ws + at * HD), *ml = (const char*)(a.ws_ml + at * 2);
  const uint32_t step = (uint32_t)(a.kv_heads * n) * 8u, step_o = step * (HD / 2);
  const int i = seq_uni(seq_div(r, a.by_group));
  const int sees = max(a.causal ? w.kvn - w.qn + i + 1 : w.kvn, 0);
  int parts = w.cut.parts;  // those the row sees
  while (parts > 0 && (parts - 1) * w.cut.part_keys >= sees) --parts;
  const uint32_t po = (uint32_t)(tid % LPR) * 16u;
  auto ml_at = [&](uint32_t off, float& pm, float& pl) {
    const u32x2 x = ld64(ml + off);
    pm = __builtin_bit_cast(float, (uint32_t)x[0]);
    pl = __builtin_bit_cast(float, (uint32_t)x[1]);
  };
  const int p0 = tid / LPR;

  float m[MLS], l[MLS];
#pragma unroll
  for (int x = 0; x < MLS; ++x) {
    const int p = lane + 64 * x;
    m[x] = NEG_INF;
    l[x] = 0.f;
    if (p < parts) ml_at(p * step, m[x], l[x]);
  }
  f32x4 o[NP];
  float om[NP], ol[NP];
  auto fetch = [&](int b) {
#pragma unroll
    for (int x = 0; x < NP; ++x) {
      const int p = b + p0 + GRP * x;
      o[x] = f32x4{0.f, 0.f, 0.f, 0.f};
      om[x] = NEG_INF;
      ol[x] = 0.f;
      if (p < parts) {
        o[x] = *reinterpret_cast<const f32x4*>(first + (po + p * step_o));
        ml_at(p * step, om[x], ol[x]);
      }
    }
  };
  fetch(0);
  float M = m[0];
#pragma unroll
  for (int x = 1; x < MLS; ++x) M = fmaxf(M, m[x]);
#pragma unroll
  for (int x = WAVE ? SEQ_WAVE_PARTS / 2 : 32; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor(M, x, 64));
  if (WAVE) M = __shfl(M, 0, 64);
  // (A part whose m is NaN makes L and the row NaN; M = -inf leaves L = 0.)
  auto weight = [&](float pm, float pl) { return pm == NEG_INF ? 0.f : pl * exp2f(pm - M); };
  float L = 0.f;
#pragma unroll
  for (int x = 0; x < MLS; ++x) L += weight(m[x], l[x]);
  L = wave_sum(L);
  // Scaled by a power of two to a sum in [1/2, 1): the same bits, and values
  // near the end of fp32's range add up within it.
  const int scale = -__builtin_amdgcn_frexp_expf(L);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int b = 0; b < parts; b += GRP * NP) {
    if (b > 0) fetch(b);
#pragma unroll
    for (int x = 0; x < NP; ++x) {
      const float f = ldexpf(weight(om[x], ol[x]), scale);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += f * o[x][e];
    }
  }
  if constexpr (WAVE) {
#pragma unroll
    for (int x = 32; x >= LPR; x >>= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], x, 64);
  } else {
    *reinterpret_cast<f32x4*>(red[tid]) = acc;
    __syncthreads();
    if (tid < LPR) {
#pragma unroll
      for (int x = 1; x < GRP; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += red[x * LPR + tid][e];
    }
    __syncthreads();  // before the next row
  }
  if (tid < LPR) {
    float out[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = L != 0.f ? acc[e] / ldexpf(L, scale) : (sees > 0 ? __builtin_nanf("") : 0.f);
    store4<T>((T*)a.o + (int64_t)(w.q0 + i) * a.o_st + (int64_t)(hk * a.group + r - i * a.group) * a.o_sh + 4 * tid, out);
  }
}

template <typename T, int HD>
__global__ __launch_bounds__(256, 4) void seq_attn_join_kernel(SeqAttnArgs a) {
  __shared__ __attribute__((aligned(16))) float red[256][4];
  const SeqShape sh = sq_shape(a);
  __shared__ int seqs[SeqWalk::LDS_INTS];
  SeqWalk walk;
  walk.init(a.s, sh, true, seqs);
  SeqWork w;
  for (int i = blockIdx.x; walk.find(a.s, sh, true, i, w); i += gridDim.x) {
    const int all = w.qn * a.heads;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // as in seq_attn_paged_kernel
    if (w.cut.parts <= SEQ_WAVE_PARTS) {
      const int u = (i - w.item) * 4 + seq_uni((int)(threadIdx.x >> 6));
      const int r = seq_uni(seq_div(u, a.by_kv_heads));
      if (u < all) sq_join_row<T, HD, true>(a, w, u - r * a.kv_heads, r, tid, red);
    } else {
      const int u = i - w.item, r = seq_uni(seq_div(u, a.by_kv_heads));
      sq_join_row<T, HD, false>(a, w, u - r * a.kv_heads, r, tid, red);
    }
  }
}

// ------------------------------------------------------------------- launch
static SeqBounds sq_bounds(const SeqAttnArgs& a) {
  return seq_bounds(sq_shape(a), a.s.tokens, a.s.batch, (int64_t)a.s.max_pages << a.s.page_log2);
}
static void sq_finish(SeqAttnArgs& a) {
  const int cus = device_cu_count();
  const SeqShape s = seq_shape(a.s.tokens, a.s.batch, a.group, a.kv_heads, a.head_dim, a.max_q_len, cus > 0 ? cus : 256);
  a.cus = s.cus;
  a.few_parts = s.few_parts;
  a.few = s.few;
}

int64_t seq_attention_workspace(const SeqAttnArgs& a0) {
  SeqAttnArgs a = a0;
  sq_finish(a);
  return sq_bounds(a).partials * (a.head_dim + 2);
}

template <typename T, int HD>
static int launch_hd(SeqAttnArgs a, hipStream_t st) {
  const dim3 block(SQ_THREADS);
  a.by_group = seq_div_by(a.group);
  a.by_kv_heads = seq_div_by(a.kv_heads);
  if (!a.paged) {
    const SeqOrder o = seq_order(a.s, a.group, SQ_ROWS, (int64_t)a.s.tokens * a.kv_heads * HD * 4);
    seq_attn_packed_kernel<T, HD><<<dim3((unsigned)seq_order_grid(o, a.kv_heads)), block, 0, st>>>(a, o);
    return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
  }
  sq_finish(a);
  const SeqBounds b = sq_bounds(a);
  a.ws_ml = a.ws + b.partials * HD;
  auto grid = [](int64_t items, int64_t most) { return dim3((unsigned)(items < most ? items : most)); };
  // As many workgroups as are resident: few rows 4 a CU at head dim 64 and 2 at
  // 128, tiles 3 and 2.
  if (a.few) seq_attn_paged_kernel<T, HD, true><<<grid(b.items, (HD == 64 ? 4 : 2) * a.cus), block, 0, st>>>(a);
  else seq_attn_paged_kernel<T, HD, false><<<grid(b.items, (HD == 64 ? 3 : 2) * a.cus), block, 0, st>>>(a);
  if (hipGetLastError() != hipSuccess) return TX_EHIP;
  if (b.partials > 0) {
    seq_attn_join_kernel<T, HD><<<grid(b.join_rows, 4 * a.cus), block, 0, st>>>(a);
    if (hipGetLastError() != hipSuccess) return TX_EHIP;
  }
  return TX_OK;
}

template <typename T>
static int launch_typed(const SeqAttnArgs& a, hipStream_t st) {
  return a.head_dim == 64 ? launch_hd<T, 64>(a, st) : launch_hd<T, 128>(a, st);
}

int launch_seq_attention(const SeqAttnArgs& a, int dt, hipStream_t st) {
  return dt == TX_BF16 ? launch_typed<bf16>(a, st) : launch_typed<f16>(a, st);
}

}  // namespace tx
