// The accepted path of a draft tree moves to the front of the drafts' slots:
//   key base + i <- key base + path[i],  i < count,  base = kv_len - n.
//
// Bound by the chain of a call's loads (starts, path, pages, rows).  A thread owns
// 16 bytes of a head's row (or a scale) and makes all moves of its sequence, so
// moves need no order between threads; a path ascends, path[i] >= i, so a slot
// that a move writes is read by no later one, and AC_AT_ONCE rows are read before
// the first of them is written.
//
// Measured: one path of 5 over 8 heads 3.3 us, a launch and the chain; 64 paths of
// up to 8 over 96 heads of 128 and 8 bits (12 layers that share pages) 7.1, 0.9
// TB/s of rows that lie 2 KB apart.  A row after another took 12.5.
#include "seq_common.hpp"

namespace tx {

constexpr int AC_THREADS = 256;
constexpr int AC_AT_ONCE = 8;

template <typename V>
__device__ __forceinline__ void ac_move(const SeqArgs& s, int b, int base, int n, int count, const int32_t* path, char* p,
                                        int64_t sp, int64_t st) {
  auto at = [&](int i) -> char* {
    if (i < 0 || i >= n) return nullptr;
    const int key = base + i, page = seq_page(s, b, key), slot = key & ((1 << s.page_log2) - 1);
    return page < 0 ? nullptr : p + page * sp + slot * st;
  };
  for (int i0 = 0; i0 < count; i0 += AC_AT_ONCE) {
    V x[AC_AT_ONCE];
    char* to[AC_AT_ONCE];
#pragma unroll
    for (int u = 0; u < AC_AT_ONCE; ++u) {
      const int i = i0 + u, f = i < count ? path[i] : -1;
      const char* from = f == i ? nullptr : at(f);
      to[u] = from ? at(i) : nullptr;
      if (to[u]) x[u] = *reinterpret_cast<const V*>(from);
    }
#pragma unroll
    for (int u = 0; u < AC_AT_ONCE; ++u)
      if (to[u]) *reinterpret_cast<V*>(to[u]) = x[u];
  }
}

__global__ __launch_bounds__(AC_THREADS) void cache_accept_kernel(CacheAcceptArgs a) {
  const int b = blockIdx.x;
  const int c0 = seq_cut(a.s.cu[b], 0, 1 << 30), n = max(seq_cut(a.s.cu[b + 1], 0, 1 << 30) - c0, 0);
  const int kvn = max(a.s.kv_lens[b], 0);
  const int count = min(max(a.counts[b], 0), min(a.max_path, n)), base = kvn - n;
  const int32_t* path = a.path + b * a.path_ld;
  int u = blockIdx.y * AC_THREADS + threadIdx.x;
  if (u == 0) a.lens_out[b] = base + count;
  const int rows = a.heads * a.chunks;
  if (u < 2 * rows) {
    const bool v = u >= rows;
    if (v) u -= rows;
    const int h = u / a.chunks, c = u - h * a.chunks;
    char* p = (char*)(v ? a.v_cache : a.k_cache) + h * (v ? a.vc_sh : a.kc_sh) + 16 * c;
    ac_move<u32x4>(a.s, b, base, n, count, path, p, v ? a.vc_sp : a.kc_sp, v ? a.vc_st : a.kc_st);
    return;
  }
  if (!a.k_scales) return;
  u -= 2 * rows;
  const int scales = a.heads * a.blocks;
  if (u >= 2 * scales) return;
  const bool v = u >= scales;
  if (v) u -= scales;
  const int h = u / a.blocks, c = u - h * a.blocks;
  char* p = (char*)(v ? a.v_scales : a.k_scales) + h * (v ? a.vs_sh : a.ks_sh) + c;
  ac_move<uint8_t>(a.s, b, base, n, count, path, p, v ? a.vs_sp : a.ks_sp, v ? a.vs_st : a.ks_st);
}

int launch_cache_accept(const CacheAcceptArgs& a, hipStream_t st) {
  const int64_t units = 2 * (int64_t)a.heads * (a.chunks + (a.k_scales ? a.blocks : 0));
  const dim3 grid((unsigned)a.s.batch, (unsigned)((units + AC_THREADS - 1) / AC_THREADS));
  cache_accept_kernel<<<grid, AC_THREADS, 0, st>>>(a);
  return hipGetLastError() == hipSuccess ? TX_OK : TX_EHIP;
}

}  // namespace tx
