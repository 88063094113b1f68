// Key and value tiles of 64 keys in LDS and their MFMA operands, shared by the
// attention kernels: 16-byte chunk swizzles, per-lane fragment offsets, the
// transposing reads of natural-layout V, and S^T = K Q^T of a tile.
#pragma once

#include "common.hpp"

namespace tx {

constexpr int AX_BN = 64;      // keys per tile

// Chunk swizzle of 128-byte LDS rows (a K tile at head dim 64, a V^T tile):
// the 16 rows one ds_read_b128 cycle serves, read at one logical chunk,
// land in 16 different 16-byte bank groups.  The hardware folds address bit
// 10 (row bit 3 here) into the bank group itself, so the row's low three
// bits are the whole swizzle.
__device__ __forceinline__ int ax_swz8(int r) { return r & 7; }
template <int HD>
__device__ __forceinline__ int ax_kswz(int key) {
  if constexpr (HD == 128) return key & 15;
  else return ax_swz8(key);
}
// Chunk swizzle of a natural-layout V tile [64 keys][HD], chosen for the
// transposed PV operand reads (ds_read_b64_tr_b16): the 32 lanes of one
// read cycle cover four consecutive keys x 64 bytes, which this XOR spreads
// over all 64 banks (checked exhaustively on the host for both head dims).
template <int HD>
__device__ __forceinline__ int ax_vswz(int key) {
  if constexpr (HD == 128) return (key & 3) << 2;
  else return ((key >> 1) & 1) << 2;
}
// Per-lane element offsets of the K fragments inside a K tile, one per
// 16-wide k step: key (lane & 31) (the t = 1 half adds 32 * HD), its
// swizzled chunk 2 ks + (lane >> 5).  Tile-independent, computed once.
template <int HD>
struct AxKOff {
  int off[HD / 16];
  __device__ __forceinline__ void init(int lane) {
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) off[ks] = col * HD + (((2 * ks + half) ^ ax_kswz<HD>(col)) << 3);
  }
  // Key-permuted operand: MFMA row i reads key i with bits 2 and 3 swapped,
  // so score slot (t, r) of lane half h holds key 32 t + 16 (r >> 3) + 8 h +
  // (r & 7).  The eight slots 8 hh .. 8 hh + 7 of a lane are then eight
  // consecutive keys in the order of a 16-key P operand (lanes 0-31: keys
  // 0-7, lanes 32-63: keys 8-15), with no cross-lane exchange.  Each group of
  // 16 lanes still reads rows 0-15 (or 16-31) as a set: same LDS banks.
  __device__ __forceinline__ void init_perm(int lane) {
    const int col = lane & 31, half = lane >> 5;
    const int row = (col & ~12) | ((col & 4) << 1) | ((col & 8) >> 1);
#pragma unroll
    for (int ks = 0; ks < HD / 16; ++ks) off[ks] = row * HD + (((2 * ks + half) ^ ax_kswz<HD>(row)) << 3);
  }
};
// Natural-layout V: per-lane element offsets of the transposed operand reads.
// The PV operand of MFMA step u and head-dim block dt gives lane l the eight
// keys 16u + 8(l >> 5) .. +7 of head-dim column 32 dt + (l & 31).  Two
// ds_read_b64_tr_b16 form it: within each 16-lane group (g = l >> 4,
// j = l & 15) result element i of lane j is element j % 4 of the 8 bytes
// addressed by lane 4 i + j / 4 (layout measured on gfx950).  So lane j
// addresses key 4r + j / 4 (+ 16u + 8(g >> 1)) at head-dim column
// 32 dt + 16 (g & 1) + 4 (j % 4) for read r: lane j receives column
// 32 dt + 16 (g & 1) + j of keys 4r .. 4r + 3.  off[dt] is the element
// offset for u = 0, r = 0; step u adds 16 u HD, read r adds 4 r HD (the
// swizzle depends on key % 4 only, which u and r leave unchanged).
template <int HD>
struct AxVNatOff {
  int off[HD / 32];
  __device__ __forceinline__ void init(int lane) {
    const int g = lane >> 4, j = lane & 15;
    const int key = 8 * (g >> 1) + (j >> 2);
#pragma unroll
    for (int dt = 0; dt < HD / 32; ++dt) {
      const int d = 32 * dt + 16 * (g & 1) + 4 * (j & 3);
      off[dt] = key * HD + (((d >> 3) ^ ax_vswz<HD>(key)) << 3) + (d & 7);
    }
  }
};

// The operand of step U at LDS byte address addr (read r = 0) and
// addr + 8 HD bytes (r = 1).  Issued from inline asm so that the key offsets
// are the instructions' immediate offsets (the builtin does not fold them,
// leaving two address instructions per read).  The compiler does not count
// these reads, so ax_vnat_wait must complete them before the operand is
// used; an uncounted LDS read can only make the compiler's own lgkmcnt waits
// stricter (LDS reads complete in order), never looser.
template <int HD, int U>
__device__ __forceinline__ u32x4 ax_vnat_issue(uint32_t addr) {
  u32x2 lo, hi;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(lo) : "v"(addr), "n"(2 * 16 * U * HD));
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(hi) : "v"(addr), "n"(2 * (16 * U * HD + 4 * HD)));
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
// Wait for every LDS read of this wave, then hand the operands on (the
// in/out operands order the wait between the reads and the MFMAs).
template <int N>
__device__ __forceinline__ void ax_vnat_wait(u32x4 (&v)[N]) {
  if constexpr (N == 2) asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v[0]), "+v"(v[1]));
  else asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
}

// S^T of one tile: s[t][r] = q_(lane&31) . k_(32t + mfma32_row(r, lane)).
// init: the accumulators' starting value (zero when null).
template <typename T, int HD>
__device__ __forceinline__ void ax_scores(const T* Ks, const typename Mfma<T>::vec* qf,
                                          const AxKOff<HD>& ko, f32x16* s, const f32x16* init = nullptr) {
  typedef typename Mfma<T>::vec vec;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[t][r] = init ? (*init)[r] : 0.f;
  // The two 32-key halves alternate: consecutive MFMAs use different
  // accumulators.
#pragma unroll
  for (int ks = 0; ks < HD / 16; ++ks) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const vec kf = *reinterpret_cast<const vec*>(Ks + 32 * t * HD + ko.off[ks]);
      s[t] = Mfma<T>::mma32(kf, qf[ks], s[t]);
    }
  }
}

}  // namespace tx
