// C-ABI entry points: host-side validation, then one launch on the caller's
// stream.  Nothing here allocates, frees or synchronises.
#include <cstdlib>
#include <mutex>

#include "tx_internal.hpp"

namespace tx {

int device_cu_count() {
  // Per-device cache; filled outside any stream capture (attribute queries
  // are not stream operations, so they are legal during capture as well).
  static int cache[64];
  static std::once_flag once[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  std::call_once(once[dev], [dev]() {
    int v = 0;
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) v = 0;
    cache[dev] = v;
  });
  return cache[dev];
}

int64_t device_shared_mem_per_block() {
  static int64_t cache[64];
  static std::once_flag once[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 0;
  std::call_once(once[dev], [dev]() {
    int v = 0;
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMaxSharedMemoryPerBlock, dev) != hipSuccess) v = 0;
    cache[dev] = v;
  });
  return cache[dev];
}

static thread_local int thread_kernel[2] = {-1, -1};  // TX_SELECT_*

int selected_kernel(int op) {
  if (thread_kernel[op] >= 0) return thread_kernel[op];
  auto env = [](const char* name) {
    const char* e = getenv(name);
    return e ? atoi(e) : -1;
  };
  static const int process_kernel[2] = {env("TX_GEMM_VARIANT"), env("TX_ATTN_ROWRES")};
  return process_kernel[op];
}

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
static inline bool is16(int dt) { return dt == TX_F16 || dt == TX_BF16; }
static inline bool isdt(int dt) { return dt == TX_F32 || dt == TX_F16 || dt == TX_BF16; }

}  // namespace tx

using namespace tx;

extern "C" {

int tx_abi_version(void) { return TX_ABI_VERSION; }

const char* tx_status_string(int code) {
  switch (code) {
    case TX_OK:
      return "ok";
    case TX_EINVAL:
      return "invalid argument (null pointer, non-positive size or bad stride)";
    case TX_EUNSUPPORTED:
      return "unsupported configuration (dtype combination, alignment or head_dim)";
    case TX_EHIP:
      return "HIP launch error";
    case TX_ESCRATCH:
      return "problem exceeds the fixed scratch buffer of the no-allocation entry point "
             "(batch * heads * seq > TX_NOALLOC_MAX_STAT_ROWS)";
    default:
      return "unknown tx status";
  }
}

int tx_device_cu_count(void) { return device_cu_count(); }

int tx_eager_softmax_supported(int64_t seq, int64_t shared_mem_per_block) {
  if (shared_mem_per_block <= 0) shared_mem_per_block = device_shared_mem_per_block();
  if (shared_mem_per_block <= 0) return -1;
  return eager_softmax_mirrorable(seq, shared_mem_per_block) ? 1 : 0;
}

int tx_select_kernel(int op, int variant) {
  if (op != TX_SELECT_GEMM && op != TX_SELECT_ATTN_ROWRES) return TX_EINVAL;
  thread_kernel[op] = variant < 0 ? -1 : variant;
  return TX_OK;
}

int tx_layernorm_residual(const void* x, const void* delta, void* x_out, void* y,
                          const void* gamma, const void* beta, const uint8_t* row_valid,
                          float* mean_out, float* rstd_out,
                          int64_t rows, int64_t d, float eps, int x_dt, int delta_dt, int y_dt,
                          int param_dt, uint32_t flags, void* stream) {
  if (!x || !y || !gamma || !beta || rows <= 0 || d <= 0 || !(eps >= 0.f)) return TX_EINVAL;
  if ((flags & TX_LN_HAS_DELTA) && !delta) return TX_EINVAL;
  if ((flags & TX_LN_WRITE_X) && !x_out) return TX_EINVAL;
  if (flags & ~63u) return TX_EINVAL;
  if (!isdt(x_dt) || !isdt(y_dt) || !isdt(param_dt)) return TX_EINVAL;
  if ((flags & TX_LN_HAS_DELTA) && delta_dt != x_dt) return TX_EUNSUPPORTED;
  if (d % 8 != 0 || d > 8192) return TX_EUNSUPPORTED;
  if (!aligned16(x) || !aligned16(y) || !aligned16(gamma) || !aligned16(beta) ||
      (delta && !aligned16(delta)) || (x_out && !aligned16(x_out)) ||
      ((uintptr_t)mean_out & 3u) || ((uintptr_t)rstd_out & 3u))
    return TX_EUNSUPPORTED;
  LayerNormArgs a{x, delta, x_out, y, gamma, beta,
                  (flags & (TX_LN_MASK_DELTA | TX_LN_MASK_X | TX_LN_MASK_OUT)) ? row_valid : nullptr,
                  mean_out, rstd_out, rows, d, eps, x_dt, y_dt, param_dt, flags};
  return launch_layernorm(a, (hipStream_t)stream);
}

int tx_gemm(const void* a, int64_t lda, const void* w, int64_t ldw, const void* bias,
            const void* residual, int64_t ldr, void* c, int64_t ldc, int64_t m, int64_t n,
            int64_t k, int ab_dt, int c_dt, int bias_dt, int res_dt, uint32_t epilogue,
            const uint8_t* row_valid, void* stream) {
  if (!a || !w || !c || m <= 0 || n <= 0 || k <= 0) return TX_EINVAL;
  if (epilogue & ~63u) return TX_EINVAL;
  if ((epilogue & TX_EPI_SPLIT_OUT) &&
      (epilogue & (TX_EPI_RESIDUAL | TX_EPI_MASK_DELTA | TX_EPI_MASK_OUT)))
    return TX_EINVAL;
  if ((epilogue & TX_EPI_SPLIT_OUT) && (ldc < 2 * n || c_dt != ab_dt)) return TX_EINVAL;
  if ((epilogue & TX_EPI_BIAS) && !bias) return TX_EINVAL;
  if ((epilogue & TX_EPI_RESIDUAL) && (!residual || ldr < n)) return TX_EINVAL;
  if (lda < k || ldw < k || ldc < n) return TX_EINVAL;
  if (m > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff) return TX_EUNSUPPORTED;
  if (!is16(ab_dt) || !isdt(c_dt) || !isdt(bias_dt) || !isdt(res_dt)) return TX_EINVAL;
  if (k % 8 || lda % 8 || ldw % 8) return TX_EUNSUPPORTED;
  if (!aligned16(a) || !aligned16(w)) return TX_EUNSUPPORTED;
  GemmArgs g{};
  g.a = a;
  g.w = w;
  g.bias = bias;
  g.res = residual;
  g.c = c;
  g.row_valid = (epilogue & (TX_EPI_MASK_DELTA | TX_EPI_MASK_OUT)) ? row_valid : nullptr;
  g.lda = lda;
  g.ldw = ldw;
  g.ldr = ldr;
  g.ldc = ldc;
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.epi = epilogue;
  return launch_gemm(g, ab_dt, c_dt, bias_dt, res_dt, false, (hipStream_t)stream);
}

int tx_qkv_proj(const void* a, const void* w_qkv, const void* b_qkv, void* qk, void* vt,
                int64_t ldvt, int64_t batch, int64_t seq, int64_t d_model, int64_t heads, int dt,
                void* stream) {
  if (!a || !w_qkv || !b_qkv || !qk || !vt) return TX_EINVAL;
  if (batch <= 0 || seq <= 0 || d_model <= 0 || heads <= 0 || d_model % heads) return TX_EINVAL;
  if (ldvt < seq) return TX_EINVAL;
  if (!is16(dt)) return TX_EUNSUPPORTED;
  if (ldvt % 8 || d_model % 64) return TX_EUNSUPPORTED;
  if (batch > 0x7fffffff || seq > 0x7fffffff || d_model > 0x7fffffff) return TX_EUNSUPPORTED;
  if (batch * seq > 0x7fffffff || 3 * d_model > 0x7fffffff || batch * heads > 0x7fffffff)
    return TX_EUNSUPPORTED;
  if (!aligned16(a) || !aligned16(w_qkv) || !aligned16(vt)) return TX_EUNSUPPORTED;
  GemmArgs g{};
  g.a = a;
  g.w = w_qkv;
  g.bias = b_qkv;
  g.c = qk;
  g.lda = d_model;
  g.ldw = d_model;
  g.ldc = 2 * d_model;
  g.m = (int)(batch * seq);
  g.n = (int)(3 * d_model);
  g.k = (int)d_model;
  g.epi = TX_EPI_BIAS;
  g.vt = vt;
  g.ldvt = ldvt;
  g.qk_cols = (int)(2 * d_model);
  g.seq = (int)seq;
  g.heads = (int)heads;
  g.head_dim = (int)(d_model / heads);
  return launch_gemm(g, dt, dt, dt, dt, true, (hipStream_t)stream);
}

int tx_flash_attn_fwd_noalloc(const void* qk, const void* vt, int64_t ldvt, void* o,
                              const uint8_t* key_valid, int64_t batch, int64_t seq, int64_t heads,
                              int64_t head_dim, float scale, int causal, int softmax_mode, int dt,
                              void* stream) {
  if (batch <= 0 || seq <= 0 || heads <= 0) return TX_EINVAL;
  if (softmax_mode != TX_SOFTMAX_EAGER)  // the online softmax uses no workspace
    return tx_flash_attn_fwd(qk, vt, ldvt, o, key_valid, batch, seq, heads, head_dim, scale, causal,
                             softmax_mode, nullptr, dt, stream);
  // Each factor is bounded first, so the products cannot overflow.
  if (batch > TX_NOALLOC_MAX_STAT_ROWS || heads > TX_NOALLOC_MAX_STAT_ROWS ||
      seq > TX_NOALLOC_MAX_STAT_ROWS || batch * heads > TX_NOALLOC_MAX_STAT_ROWS ||
      batch * heads * seq > TX_NOALLOC_MAX_STAT_ROWS)
    return TX_ESCRATCH;
  float* stats = scratch_device_ptr();
  if (!stats) return TX_EHIP;
  return tx_flash_attn_fwd(qk, vt, ldvt, o, key_valid, batch, seq, heads, head_dim, scale, causal,
                           softmax_mode, stats, dt, stream);
}

int tx_flash_attn_fwd(const void* qk, const void* vt, int64_t ldvt, void* o,
                      const uint8_t* key_valid, int64_t batch, int64_t seq, int64_t heads,
                      int64_t head_dim, float scale, int causal, int softmax_mode,
                      float* row_stats, int dt, void* stream) {
  if (!qk || !vt || !o) return TX_EINVAL;
  if (batch <= 0 || seq <= 0 || heads <= 0 || head_dim <= 0 || ldvt < seq) return TX_EINVAL;
  if (!(scale > 0.f) || !(scale < 3.0e38f)) return TX_EINVAL;
  if (softmax_mode != TX_SOFTMAX_EAGER && softmax_mode != TX_SOFTMAX_ONLINE) return TX_EINVAL;
  if (softmax_mode == TX_SOFTMAX_EAGER && (!row_stats || ((uintptr_t)row_stats & 7u)))
    return TX_EINVAL;
  if (!is16(dt)) return TX_EUNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return TX_EUNSUPPORTED;
  if (ldvt % 8) return TX_EUNSUPPORTED;
  if (batch > 0x7fffffff || seq > 0x7fffffff || heads > 0x7fffffff) return TX_EUNSUPPORTED;
  if (batch * seq > 0x7fffffff || batch * heads > 0x7fffffff) return TX_EUNSUPPORTED;
  if (!aligned16(qk) || !aligned16(vt) || ((uintptr_t)o & 7u)) return TX_EUNSUPPORTED;
  // The packed layouts as strided views: q = qk[:, :D], k = qk[:, D:],
  // heads at stride head_dim; V^T rows of ldvt keys; o = [B*S, D].
  const int64_t d = heads * head_dim;
  // The K and V^T tile loaders form per-lane byte offsets within a tile in
  // 32 bits: 64 key rows of 2D elements, head_dim V^T rows of ldvt.
  if (d >= (int64_t)1 << 24 || head_dim * ldvt * 2 + 256 > (int64_t)0xffffffff) return TX_EUNSUPPORTED;
  // o is written while other workgroups still read q, k and v.
  {
    const int64_t qk_bytes = batch * seq * 2 * d * 2, vt_bytes = batch * heads * head_dim * ldvt * 2;
    const int64_t o_bytes = batch * seq * d * 2;
    if (spans_overlap((uintptr_t)o, o_bytes, (uintptr_t)qk, qk_bytes) ||
        spans_overlap((uintptr_t)o, o_bytes, (uintptr_t)vt, vt_bytes))
      return TX_EINVAL;
  }
  AttnArgs at{};
  at.q = qk;
  at.k = (const char*)qk + d * 2;  // 16-bit elements
  at.v = vt;
  at.o = o;
  at.q_sb = at.k_sb = seq * 2 * d;
  at.q_sh = at.k_sh = head_dim;
  at.q_ss = at.k_ss = 2 * d;
  at.v_sb = heads * head_dim * ldvt;
  at.v_sh = head_dim * ldvt;
  at.v_ss = 0;
  at.o_sb = seq * d;
  at.o_sh = head_dim;
  at.o_ss = d;
  at.key_valid = key_valid;
  at.kv_sb = seq;
  at.vnat = 0;
  at.ldvt = ldvt;
  at.batch = (int)batch;
  at.seq = (int)seq;
  at.heads = (int)heads;
  at.head_dim = (int)head_dim;
  at.scale = scale;
  at.causal = causal ? 1 : 0;
  at.softmax_mode = softmax_mode;
  at.row_stats = row_stats;
  return launch_attention(at, dt, (hipStream_t)stream);
}

int tx_flash_attn_fwd_strided(const void* q, const void* k, const void* v, void* o,
                              const int64_t* q_strides, const int64_t* k_strides,
                              const int64_t* v_strides, const int64_t* o_strides,
                              const uint8_t* key_valid, int64_t key_valid_sb, int64_t batch,
                              int64_t heads, int64_t seq, int64_t head_dim, float scale, int causal,
                              int softmax_mode, float* row_stats, int dt, void* stream) {
  if (!q || !k || !v || !o || !q_strides || !k_strides || !v_strides || !o_strides) return TX_EINVAL;
  if (batch <= 0 || seq <= 0 || heads <= 0 || head_dim <= 0) return TX_EINVAL;
  if (!(scale > 0.f) || !(scale < 3.0e38f)) return TX_EINVAL;
  if (softmax_mode != TX_SOFTMAX_EAGER && softmax_mode != TX_SOFTMAX_ONLINE) return TX_EINVAL;
  if (softmax_mode == TX_SOFTMAX_EAGER && (!row_stats || ((uintptr_t)row_stats & 7u)))
    return TX_EINVAL;
  if (key_valid && key_valid_sb < seq) return TX_EINVAL;
  const int64_t* in_strides[3] = {q_strides, k_strides, v_strides};
  for (int t = 0; t < 3; ++t) {
    const int64_t* st = in_strides[t];
    if (st[0] < 0 || st[1] < 0 || st[2] < 0) return TX_EINVAL;
    if (st[3] != 1) return TX_EUNSUPPORTED;  // head_dim must be contiguous
    // 16-byte rows for the 128-bit loads and the DMA; row offsets of a tile
    // are 32-bit byte offsets (64 rows).
    if (st[0] % 8 || st[1] % 8 || st[2] % 8 || st[2] >= (1 << 24)) return TX_EUNSUPPORTED;
  }
  if (o_strides[0] < 0 || o_strides[1] < 0 || o_strides[2] < head_dim) return TX_EINVAL;
  if (o_strides[3] != 1 || o_strides[0] % 4 || o_strides[1] % 4 || o_strides[2] % 4)
    return TX_EUNSUPPORTED;
  if (!is16(dt)) return TX_EUNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return TX_EUNSUPPORTED;
  if (batch > 0x7fffffff || seq > 0x7fffffff || heads > 0x7fffffff) return TX_EUNSUPPORTED;
  if (batch * seq > 0x7fffffff || batch * heads > 0x7fffffff) return TX_EUNSUPPORTED;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || ((uintptr_t)o & 7u)) return TX_EUNSUPPORTED;
  // Every (b, h, s) output row is written by one workgroup: distinct rows
  // may not share elements (o_strides[1] = 0 would make every head's
  // workgroups race on one row), and o may not share memory with q, k or v,
  // which other workgroups still read while it is written.
  if (!view_is_nonoverlapping(o_strides, batch, heads, seq, head_dim)) return TX_EINVAL;
  {
    const int64_t* views[4] = {q_strides, k_strides, v_strides, o_strides};
    const void* ptrs[4] = {q, k, v, o};
    int64_t bytes[4];
    for (int t = 0; t < 4; ++t) {
      const int64_t mo = view_max_offset(views[t], batch, heads, seq, head_dim);
      if (mo < 0) return TX_EUNSUPPORTED;
      bytes[t] = (mo + 1) * 2;
    }
    for (int t = 0; t < 3; ++t)
      if (spans_overlap((uintptr_t)o, bytes[3], (uintptr_t)ptrs[t], bytes[t])) return TX_EINVAL;
  }
  AttnArgs at{};
  at.q = q;
  at.k = k;
  at.v = v;
  at.o = o;
  at.q_sb = q_strides[0];
  at.q_sh = q_strides[1];
  at.q_ss = q_strides[2];
  at.k_sb = k_strides[0];
  at.k_sh = k_strides[1];
  at.k_ss = k_strides[2];
  at.v_sb = v_strides[0];
  at.v_sh = v_strides[1];
  at.v_ss = v_strides[2];
  at.o_sb = o_strides[0];
  at.o_sh = o_strides[1];
  at.o_ss = o_strides[2];
  at.key_valid = key_valid;
  at.kv_sb = key_valid_sb;
  at.vnat = 1;
  at.ldvt = 0;
  at.batch = (int)batch;
  at.seq = (int)seq;
  at.heads = (int)heads;
  at.head_dim = (int)head_dim;
  at.scale = scale;
  at.causal = causal ? 1 : 0;
  at.softmax_mode = softmax_mode;
  at.row_stats = row_stats;
  return launch_attention(at, dt, (hipStream_t)stream);
}

// ---- packed sequences and the paged cache ------------------------------------
// A [rows][heads][head_dim] view: 16-byte rows, heads that do not overlap, and
// (outputs) rows that do not either.
static int check_rows(const void* p, const int64_t* st, int64_t rows, int64_t heads, int64_t hd, bool out) {
  if (!p || !st) return TX_EINVAL;
  if (st[0] < 0 || st[1] < 0) return TX_EINVAL;
  if (!aligned16(p) || st[0] % 8 || st[1] % 8) return TX_EUNSUPPORTED;
  if (st[0] > (int64_t)1 << 40 || st[1] > (int64_t)1 << 40) return TX_EUNSUPPORTED;
  const int64_t st3[3] = {st[0], st[1], 0};
  if (out && !view_is_nonoverlapping(st3, rows, heads, 1, hd)) return TX_EINVAL;
  return TX_OK;
}
// A [pages][heads][slots][head_dim] cache view of elements of `size` bytes.
static int check_cache(const void* p, const int64_t* st, int64_t pages, int64_t heads, int64_t slots, int64_t hd,
                       int size = 2) {
  if (!p || !st) return TX_EINVAL;
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0) return TX_EINVAL;
    if (st[i] % (16 / size) || st[i] > (int64_t)1 << 40) return TX_EUNSUPPORTED;
  }
  if (!aligned16(p)) return TX_EUNSUPPORTED;
  // Byte strides of a page, and byte offsets within one K/V head's part of it, are 32-bit.
  if (st[2] >= 1 << 24 || st[0] >= (int64_t)1 << 31 || (slots - 1) * st[2] + hd >= (int64_t)1 << 31)
    return TX_EUNSUPPORTED;
  return view_is_nonoverlapping(st, pages, heads, slots, hd) ? TX_OK : TX_EINVAL;
}
// Scales of an 8-bit cache, [pages][heads][slots][n], rows aligned to `align` bytes.
static int check_scales(const void* p, const int64_t* st, int64_t pages, int64_t heads, int64_t slots, int64_t n,
                        int64_t align) {
  if (!p || !st) return TX_EINVAL;
  for (int i = 0; i < 3; ++i) {
    if (st[i] < 0) return TX_EINVAL;
    if (st[i] % align || st[i] > (int64_t)1 << 40) return TX_EUNSUPPORTED;
  }
  if ((uintptr_t)p % (uintptr_t)align) return TX_EUNSUPPORTED;
  if (st[2] >= 1 << 24 || st[0] >= (int64_t)1 << 31 || (slots - 1) * st[2] + n >= (int64_t)1 << 31)
    return TX_EUNSUPPORTED;
  return view_is_nonoverlapping(st, pages, heads, slots, n) ? TX_OK : TX_EINVAL;
}
// Memory that a call reads or writes: `count` blocks of `extent` bytes, `stride` apart.
struct Mem {
  uintptr_t p;
  __int128 stride, extent;
  int64_t count;
};
static Mem mem_rows(const void* p, const int64_t* st, int64_t rows, int64_t heads, int64_t hd) {
  return {(uintptr_t)p, (__int128)st[0] * 2, (__int128)((heads - 1) * st[1] + hd) * 2, rows};
}
static Mem mem_pages(const void* p, const int64_t* st, int64_t pages, int64_t heads, int64_t slots, int64_t n, int size) {
  return {(uintptr_t)p, (__int128)st[0] * size, (__int128)((heads - 1) * st[1] + (slots - 1) * st[2] + n) * size, pages};
}
static Mem mem_span(const void* p, int64_t bytes) { return {(uintptr_t)p, bytes, bytes, 1}; }
static bool disjoint(const Mem& a, const Mem& b) {
  if (!a.p || !b.p || a.extent <= 0 || b.extent <= 0) return true;
  return byte_blocks_disjoint(a.p, a.stride, a.extent, a.count, b.p, b.stride, b.extent, b.count);
}
static bool rows_disjoint(const void* a, const int64_t* as, int64_t ah, const void* b, const int64_t* bs,
                          int64_t bh, int64_t rows, int64_t hd) {
  return blocks_disjoint((uintptr_t)a, as[0], (ah - 1) * as[1] + hd, rows, (uintptr_t)b, bs[0],
                         (bh - 1) * bs[1] + hd, rows);
}
static int64_t page_extent(const int64_t* st, int64_t heads, int64_t slots, int64_t hd) {
  return (heads - 1) * st[1] + (slots - 1) * st[2] + hd;
}
static bool same_rows(const void* a, const int64_t* as, const void* b, const int64_t* bs) {
  return a == b && as[0] == bs[0] && as[1] == bs[1];
}
// Totals every entry point of this group shares.
static int check_seqs(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t hd, int dt,
                      const int32_t* cu) {
  if (!cu || tokens <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || hd <= 0) return TX_EINVAL;
  if (!is16(dt)) return TX_EUNSUPPORTED;
  if (heads % kv_heads) return TX_EINVAL;
  // Grids (256 threads per 128 rows, per 4 tokens and per sequence) stay below 2^32 threads, and the items of
  // a paged call (per 16 rows and per sequence, up to 256 parts of the keys) below 2^31.
  if (tokens > 1 << 24 || batch > 1 << 20 || heads > 65535 || tokens * heads > 1 << 26 ||
      batch * kv_heads > 1 << 23)
    return TX_EUNSUPPORTED;
  if (((uintptr_t)cu & 3u)) return TX_EUNSUPPORTED;
  return TX_OK;
}
static int check_pages(const int32_t* table, int64_t table_ld, int64_t batch, int64_t num_pages, int64_t page_size,
                       int64_t max_pages) {
  if (!table || num_pages <= 0 || page_size <= 0 || max_pages <= 0) return TX_EINVAL;
  if (batch > 1 && table_ld < max_pages) return TX_EINVAL;
  if (((uintptr_t)table & 3u) || table_ld < 0 || table_ld > (int64_t)1 << 40) return TX_EUNSUPPORTED;
  if (page_size < 8 || page_size > 1 << 15 || (page_size & (page_size - 1))) return TX_EUNSUPPORTED;
  if (num_pages > 0x7fffffff || max_pages > (int64_t)1 << 30 || max_pages * page_size > (int64_t)1 << 30)
    return TX_EUNSUPPORTED;
  return TX_OK;
}
static int page_log2(int64_t page_size) {
  int n = 0;
  while (((int64_t)1 << n) < page_size) ++n;
  return n;
}

int tx_rotary_append(const void* q, const int64_t q_strides[2], void* q_out, const int64_t q_out_strides[2],
                     const void* k, const int64_t k_strides[2], void* k_out, const int64_t k_out_strides[2],
                     const void* v, const int64_t v_strides[2], void* k_cache,
                     const int64_t k_cache_strides[3], void* v_cache, const int64_t v_cache_strides[3],
                     const int64_t* steps, const int64_t* positions, const int32_t* cu_seqlens,
                     const int32_t* kv_lens, const int32_t* block_table, int64_t table_ld, int64_t tokens,
                     int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
                     int64_t num_pages, int64_t page_size, int64_t max_pages, float amplitude, int interleaved,
                     int dt, void* stream) {
  if (!k || !steps || (!q) != (!q_out) || (!k_cache) != (!v_cache)) return TX_EINVAL;
  if (!k_out && !k_cache) return TX_EINVAL;
  if (!(amplitude > 0.f) || !(amplitude < 3.0e38f)) return TX_EINVAL;
  int rc = check_seqs(tokens, batch, q_heads, kv_heads, head_dim, dt, cu_seqlens);
  if (rc != TX_OK) return rc;
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim) return TX_EINVAL;
  if (head_dim % 8 || head_dim > 256) return TX_EUNSUPPORTED;
  if (((uintptr_t)steps & 7u) || ((uintptr_t)positions & 7u) || ((uintptr_t)kv_lens & 3u)) return TX_EUNSUPPORTED;
  // Work units of one workgroup's tokens are counted in 32 bits.
  if ((q_heads + 2 * kv_heads) * head_dim > (int64_t)1 << 26) return TX_EUNSUPPORTED;
  if (q && (rc = check_rows(q, q_strides, tokens, q_heads, head_dim, false)) != TX_OK) return rc;
  if (q && (rc = check_rows(q_out, q_out_strides, tokens, q_heads, head_dim, true)) != TX_OK) return rc;
  if ((rc = check_rows(k, k_strides, tokens, kv_heads, head_dim, false)) != TX_OK) return rc;
  if (k_out && (rc = check_rows(k_out, k_out_strides, tokens, kv_heads, head_dim, true)) != TX_OK) return rc;
  if (k_cache) {
    if (!kv_lens) return TX_EINVAL;
    if ((rc = check_rows(v, v_strides, tokens, kv_heads, head_dim, false)) != TX_OK) return rc;
    if ((rc = check_pages(block_table, table_ld, batch, num_pages, page_size, max_pages)) != TX_OK) return rc;
    if ((rc = check_cache(k_cache, k_cache_strides, num_pages, kv_heads, page_size, head_dim)) != TX_OK) return rc;
    if ((rc = check_cache(v_cache, v_cache_strides, num_pages, kv_heads, page_size, head_dim)) != TX_OK) return rc;
  }
  // Outputs: an input itself, or memory that no input and no other output uses.
  struct View {
    const void* p;
    const int64_t* st;
    int64_t extent, count;
    int in_place;  // the input (index) that it may be
  } in[3], out[4];
  int n_in = 0, n_out = 0;
  const int64_t qx = q ? (q_heads - 1) * q_strides[1] + head_dim : 0;
  const int64_t kx = (kv_heads - 1) * k_strides[1] + head_dim;
  in[n_in++] = {k, k_strides, kx, tokens, -1};
  if (q) in[n_in++] = {q, q_strides, qx, tokens, -1};
  if (k_cache) in[n_in++] = {v, v_strides, (kv_heads - 1) * v_strides[1] + head_dim, tokens, -1};
  if (k_out) out[n_out++] = {k_out, k_out_strides, (kv_heads - 1) * k_out_strides[1] + head_dim, tokens, 0};
  if (q) out[n_out++] = {q_out, q_out_strides, (q_heads - 1) * q_out_strides[1] + head_dim, tokens, 1};
  if (k_cache) {
    out[n_out++] = {k_cache, k_cache_strides, page_extent(k_cache_strides, kv_heads, page_size, head_dim), num_pages, -1};
    out[n_out++] = {v_cache, v_cache_strides, page_extent(v_cache_strides, kv_heads, page_size, head_dim), num_pages, -1};
  }
  for (int o = 0; o < n_out; ++o) {
    for (int i = 0; i < n_in; ++i) {
      if (out[o].in_place == i && same_rows(out[o].p, out[o].st, in[i].p, in[i].st)) continue;
      if (!blocks_disjoint((uintptr_t)out[o].p, out[o].st[0], out[o].extent, out[o].count, (uintptr_t)in[i].p,
                           in[i].st[0], in[i].extent, in[i].count))
        return TX_EINVAL;
    }
    for (int i = 0; i < o; ++i)
      if (!blocks_disjoint((uintptr_t)out[o].p, out[o].st[0], out[o].extent, out[o].count, (uintptr_t)out[i].p,
                           out[i].st[0], out[i].extent, out[i].count))
        return TX_EINVAL;
  }
  RotaryArgs a{};
  a.s = {cu_seqlens, kv_lens, block_table, table_ld, (int)tokens, (int)batch, 0, 0, 0};
  a.k = k;
  a.k_st = k_strides[0];
  a.k_sh = k_strides[1];
  if (q) {
    a.q = q;
    a.q_st = q_strides[0];
    a.q_sh = q_strides[1];
    a.q_out = q_out;
    a.qo_st = q_out_strides[0];
    a.qo_sh = q_out_strides[1];
  }
  if (k_out) {
    a.k_out = k_out;
    a.ko_st = k_out_strides[0];
    a.ko_sh = k_out_strides[1];
  }
  if (k_cache) {
    a.s.num_pages = (int)num_pages;
    a.s.page_log2 = page_log2(page_size);
    a.s.max_pages = (int)max_pages;
    a.v = v;
    a.v_st = v_strides[0];
    a.v_sh = v_strides[1];
    a.k_cache = k_cache;
    a.kc_sp = k_cache_strides[0];
    a.kc_sh = k_cache_strides[1];
    a.kc_st = k_cache_strides[2];
    a.v_cache = v_cache;
    a.vc_sp = v_cache_strides[0];
    a.vc_sh = v_cache_strides[1];
    a.vc_st = v_cache_strides[2];
  }
  a.steps = (const uint64_t*)steps;
  a.positions = positions;
  a.heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.head_dim = (int)head_dim;
  a.rotary = (int)rotary_dim;
  a.amplitude = amplitude;
  a.interleaved = interleaved ? 1 : 0;
  return launch_rotary_append(a, dt, (hipStream_t)stream);
}

int tx_flash_attn_packed(const void* q, const int64_t q_strides[2], const void* k, const int64_t k_strides[2],
                         const void* v, const int64_t v_strides[2], void* o, const int64_t o_strides[2],
                         const int32_t* cu_seqlens, int64_t tokens, int64_t batch, int64_t q_heads,
                         int64_t kv_heads, int64_t head_dim, float scale, int causal, int dt, void* stream) {
  int rc = check_seqs(tokens, batch, q_heads, kv_heads, head_dim, dt, cu_seqlens);
  if (rc != TX_OK) return rc;
  if (!(scale > 0.f) || !(scale < 3.0e38f)) return TX_EINVAL;
  if (head_dim != 64 && head_dim != 128) return TX_EUNSUPPORTED;
  if ((rc = check_rows(q, q_strides, tokens, q_heads, head_dim, false)) != TX_OK) return rc;
  if ((rc = check_rows(k, k_strides, tokens, kv_heads, head_dim, false)) != TX_OK) return rc;
  if ((rc = check_rows(v, v_strides, tokens, kv_heads, head_dim, false)) != TX_OK) return rc;
  if ((rc = check_rows(o, o_strides, tokens, q_heads, head_dim, true)) != TX_OK) return rc;
  // The tile loaders form 32-bit byte offsets within a tile of key rows.
  if (k_strides[0] >= 1 << 24 || v_strides[0] >= 1 << 24) return TX_EUNSUPPORTED;
  if (!rows_disjoint(o, o_strides, q_heads, q, q_strides, q_heads, tokens, head_dim) ||
      !rows_disjoint(o, o_strides, q_heads, k, k_strides, kv_heads, tokens, head_dim) ||
      !rows_disjoint(o, o_strides, q_heads, v, v_strides, kv_heads, tokens, head_dim))
    return TX_EINVAL;
  SeqAttnArgs a{};
  a.s = {cu_seqlens, nullptr, nullptr, 0, (int)tokens, (int)batch, 0, 0, 0};
  a.q = q;
  a.k = k;
  a.v = v;
  a.o = o;
  a.q_st = q_strides[0];
  a.q_sh = q_strides[1];
  a.k_st = k_strides[0];
  a.k_sh = k_strides[1];
  a.v_st = v_strides[0];
  a.v_sh = v_strides[1];
  a.o_st = o_strides[0];
  a.o_sh = o_strides[1];
  a.heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.head_dim = (int)head_dim;
  a.scale = scale;
  a.causal = causal ? 1 : 0;
  return launch_seq_attention(a, dt, (hipStream_t)stream);
}

static int paged_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t head_dim,
                           int64_t page_size, int64_t max_pages, int64_t max_q_len, bool cache, int64_t* floats) {
  const int32_t some = 0;
  int rc = check_seqs(tokens, batch, q_heads, kv_heads, head_dim, TX_BF16, &some);
  if (rc != TX_OK) return rc;
  if (!floats) return TX_EINVAL;
  if (head_dim != 64 && head_dim != 128) return TX_EUNSUPPORTED;
  if ((rc = check_pages(&some, max_pages, batch, 1, page_size, max_pages)) != TX_OK) return rc;
  SeqAttnArgs a{};
  a.s.tokens = (int)tokens;
  a.s.batch = (int)batch;
  a.s.page_log2 = page_log2(page_size);
  a.s.max_pages = (int)max_pages;
  a.heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.head_dim = (int)head_dim;
  a.paged = 1;
  a.max_q_len = max_q_len <= 0 || max_q_len > tokens ? tokens : max_q_len;
  *floats = cache ? cache_attention_workspace(a) : seq_attention_workspace(a);
  return TX_OK;
}

int tx_flash_attn_paged_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                  int64_t head_dim, int64_t page_size, int64_t max_pages, int64_t max_q_len,
                                  int64_t* floats) {
  return paged_workspace(tokens, batch, q_heads, kv_heads, head_dim, page_size, max_pages, max_q_len, false, floats);
}

int tx_flash_attn_cache_workspace(int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                                  int64_t head_dim, int64_t page_size, int64_t max_pages, int64_t max_q_len,
                                  int64_t* floats) {
  return paged_workspace(tokens, batch, q_heads, kv_heads, head_dim, page_size, max_pages, max_q_len, true, floats);
}

// What the paged calls share.  Scales (nullptr: 16-bit caches), and a tree's mask.
struct PagedExtra {
  const uint8_t* k_scales;
  const int64_t* k_scales_strides;
  const uint8_t* v_scales;
  const int64_t* v_scales_strides;
  const int64_t* tree;
  int64_t tree_ld, tree_words;
};
static int paged_attention(const void* q, const int64_t q_strides[2], const void* k_cache,
                           const int64_t k_cache_strides[3], const void* v_cache, const int64_t v_cache_strides[3],
                           void* o, const int64_t o_strides[2], const int32_t* cu_seqlens, const int32_t* kv_lens,
                           const int32_t* block_table, int64_t table_ld, int64_t tokens, int64_t batch,
                           int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size,
                           int64_t max_pages, int64_t max_q_len, float scale, int causal, float* workspace,
                           int64_t workspace_floats, int dt, const PagedExtra& x, bool mx, bool tree, void* stream) {
  int rc = check_seqs(tokens, batch, q_heads, kv_heads, head_dim, dt, cu_seqlens);
  if (rc != TX_OK) return rc;
  if (!kv_lens || !(scale > 0.f) || !(scale < 3.0e38f)) return TX_EINVAL;
  if ((uintptr_t)kv_lens & 3u) return TX_EUNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return TX_EUNSUPPORTED;
  if ((rc = check_rows(q, q_strides, tokens, q_heads, head_dim, false)) != TX_OK) return rc;
  if ((rc = check_rows(o, o_strides, tokens, q_heads, head_dim, true)) != TX_OK) return rc;
  if ((rc = check_pages(block_table, table_ld, batch, num_pages, page_size, max_pages)) != TX_OK) return rc;
  const int size = mx ? 1 : 2;
  const int64_t blocks = head_dim / 32;
  if ((rc = check_cache(k_cache, k_cache_strides, num_pages, kv_heads, page_size, head_dim, size)) != TX_OK) return rc;
  if ((rc = check_cache(v_cache, v_cache_strides, num_pages, kv_heads, page_size, head_dim, size)) != TX_OK) return rc;
  if (mx) {
    if ((rc = check_scales(x.k_scales, x.k_scales_strides, num_pages, kv_heads, page_size, blocks, blocks)) != TX_OK) return rc;
    if ((rc = check_scales(x.v_scales, x.v_scales_strides, num_pages, kv_heads, page_size, blocks, blocks)) != TX_OK) return rc;
  }
  if (tree) {
    if (!x.tree || x.tree_words <= 0 || x.tree_ld < 0 || (tokens > 1 && x.tree_ld < x.tree_words)) return TX_EINVAL;
    if (((uintptr_t)x.tree & 7u) || x.tree_words > 1 << 24 || x.tree_ld > (int64_t)1 << 40) return TX_EUNSUPPORTED;
  }
  SeqAttnArgs a{};
  a.s = {cu_seqlens, kv_lens, block_table, table_ld, (int)tokens, (int)batch, (int)num_pages,
         page_log2(page_size), (int)max_pages};
  a.q = q;
  a.k = k_cache;
  a.v = v_cache;
  a.o = o;
  a.q_st = q_strides[0];
  a.q_sh = q_strides[1];
  a.o_st = o_strides[0];
  a.o_sh = o_strides[1];
  a.k_sp = k_cache_strides[0];
  a.k_sh = k_cache_strides[1];
  a.k_st = k_cache_strides[2];
  a.v_sp = v_cache_strides[0];
  a.v_sh = v_cache_strides[1];
  a.v_st = v_cache_strides[2];
  a.heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.group = (int)(q_heads / kv_heads);
  a.head_dim = (int)head_dim;
  a.scale = scale;
  a.causal = causal ? 1 : 0;
  a.paged = 1;
  a.max_q_len = max_q_len <= 0 || max_q_len > tokens ? tokens : max_q_len;
  a.ws = workspace;
  if (mx) {
    a.k_scales = x.k_scales;
    a.v_scales = x.v_scales;
    a.ks_sp = x.k_scales_strides[0];
    a.ks_sh = x.k_scales_strides[1];
    a.ks_st = x.k_scales_strides[2];
    a.vs_sp = x.v_scales_strides[0];
    a.vs_sh = x.v_scales_strides[1];
    a.vs_st = x.v_scales_strides[2];
  }
  if (tree) {
    a.tree = (const uint64_t*)x.tree;
    a.tree_ld = x.tree_ld;
    a.tree_words = (int)x.tree_words;
  }
  const int64_t need = mx || tree ? cache_attention_workspace(a) : seq_attention_workspace(a);
  if (need > 0 && (!workspace || !aligned16(workspace) || workspace_floats < need)) return TX_EINVAL;
  // Output and workspace are written while the inputs are read.
  const Mem out = mem_rows(o, o_strides, tokens, q_heads, head_dim);
  const Mem in[] = {mem_rows(q, q_strides, tokens, q_heads, head_dim),
                    mem_pages(k_cache, k_cache_strides, num_pages, kv_heads, page_size, head_dim, size),
                    mem_pages(v_cache, v_cache_strides, num_pages, kv_heads, page_size, head_dim, size)};
  for (const Mem& m : in)
    if (!disjoint(out, m)) return TX_EINVAL;
  const Mem small[] = {mem_span(cu_seqlens, (batch + 1) * 4), mem_span(kv_lens, batch * 4),
                       mem_span(block_table, ((batch - 1) * table_ld + max_pages) * 4),
                       tree ? Mem{(uintptr_t)x.tree, (__int128)x.tree_ld * 8, (__int128)x.tree_words * 8, tokens} : Mem{},
                       mx ? mem_pages(x.k_scales, x.k_scales_strides, num_pages, kv_heads, page_size, blocks, 1) : Mem{},
                       mx ? mem_pages(x.v_scales, x.v_scales_strides, num_pages, kv_heads, page_size, blocks, 1) : Mem{}};
  if (mx || tree)
    for (const Mem& m : small)
      if (!disjoint(out, m)) return TX_EINVAL;
  if (need > 0) {
    const uintptr_t ws = (uintptr_t)workspace;
    if (span_meets_byte_blocks(ws, need * 4, out.p, out.stride, out.extent, out.count)) return TX_EINVAL;
    for (const Mem& m : in)
      if (span_meets_byte_blocks(ws, need * 4, m.p, m.stride, m.extent, m.count)) return TX_EINVAL;
    for (const Mem& m : small)
      if (m.p && span_meets_byte_blocks(ws, need * 4, m.p, m.stride, m.extent, m.count)) return TX_EINVAL;
  }
  return mx || tree ? launch_cache_attention(a, dt, (hipStream_t)stream) : launch_seq_attention(a, dt, (hipStream_t)stream);
}

int tx_flash_attn_paged(const void* q, const int64_t q_strides[2], const void* k_cache,
                        const int64_t k_cache_strides[3], const void* v_cache,
                        const int64_t v_cache_strides[3], void* o, const int64_t o_strides[2],
                        const int32_t* cu_seqlens, const int32_t* kv_lens, const int32_t* block_table,
                        int64_t table_ld, int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                        int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages,
                        int64_t max_q_len, float scale, int causal, float* workspace, int64_t workspace_floats,
                        int dt, void* stream) {
  return paged_attention(q, q_strides, k_cache, k_cache_strides, v_cache, v_cache_strides, o, o_strides, cu_seqlens, kv_lens,
                         block_table, table_ld, tokens, batch, q_heads, kv_heads, head_dim, num_pages, page_size, max_pages,
                         max_q_len, scale, causal, workspace, workspace_floats, dt, PagedExtra{}, false, false, stream);
}

int tx_flash_attn_paged_mx8(const void* q, const int64_t q_strides[2], const void* k_cache,
                            const int64_t k_cache_strides[3], const uint8_t* k_scales,
                            const int64_t k_scales_strides[3], const void* v_cache,
                            const int64_t v_cache_strides[3], const uint8_t* v_scales,
                            const int64_t v_scales_strides[3], void* o, const int64_t o_strides[2],
                            const int32_t* cu_seqlens, const int32_t* kv_lens, const int32_t* block_table,
                            int64_t table_ld, int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                            int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages,
                            int64_t max_q_len, float scale, int causal, float* workspace, int64_t workspace_floats,
                            int dt, void* stream) {
  const PagedExtra x{k_scales, k_scales_strides, v_scales, v_scales_strides, nullptr, 0, 0};
  return paged_attention(q, q_strides, k_cache, k_cache_strides, v_cache, v_cache_strides, o, o_strides, cu_seqlens, kv_lens,
                         block_table, table_ld, tokens, batch, q_heads, kv_heads, head_dim, num_pages, page_size, max_pages,
                         max_q_len, scale, causal, workspace, workspace_floats, dt, x, true, false, stream);
}

int tx_flash_attn_tree(const void* q, const int64_t q_strides[2], const void* k_cache,
                       const int64_t k_cache_strides[3], const uint8_t* k_scales,
                       const int64_t k_scales_strides[3], const void* v_cache, const int64_t v_cache_strides[3],
                       const uint8_t* v_scales, const int64_t v_scales_strides[3], void* o,
                       const int64_t o_strides[2], const int32_t* cu_seqlens, const int32_t* kv_lens,
                       const int32_t* block_table, int64_t table_ld, const int64_t* tree_mask, int64_t tree_ld,
                       int64_t tree_words, int64_t tokens, int64_t batch, int64_t q_heads, int64_t kv_heads,
                       int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages,
                       int64_t max_q_len, float scale, float* workspace, int64_t workspace_floats, int dt,
                       void* stream) {
  if ((!k_scales) != (!v_scales)) return TX_EINVAL;
  const PagedExtra x{k_scales, k_scales_strides, v_scales, v_scales_strides, tree_mask, tree_ld, tree_words};
  return paged_attention(q, q_strides, k_cache, k_cache_strides, v_cache, v_cache_strides, o, o_strides, cu_seqlens, kv_lens,
                         block_table, table_ld, tokens, batch, q_heads, kv_heads, head_dim, num_pages, page_size, max_pages,
                         max_q_len, scale, 0, workspace, workspace_floats, dt, x, k_scales != nullptr, true, stream);
}

int tx_norm_rotary_append(const void* q, const int64_t q_strides[2], void* q_out, const int64_t q_out_strides[2],
                          const void* k, const int64_t k_strides[2], void* k_out, const int64_t k_out_strides[2],
                          const void* v, const int64_t v_strides[2], void* k_cache,
                          const int64_t k_cache_strides[3], uint8_t* k_scales, const int64_t k_scales_strides[3],
                          void* v_cache, const int64_t v_cache_strides[3], uint8_t* v_scales,
                          const int64_t v_scales_strides[3], const void* q_weight, const void* q_bias,
                          const void* k_weight, const void* k_bias, int per_head, int param_dt, int norm, float eps,
                          const int64_t* steps, const int32_t* pair_axis, const int64_t* positions,
                          int64_t positions_ld, int64_t axes, const int32_t* cu_seqlens, const int32_t* kv_lens,
                          const int32_t* block_table, int64_t table_ld, int64_t tokens, int64_t batch,
                          int64_t q_heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim, int64_t num_pages,
                          int64_t page_size, int64_t max_pages, float amplitude, int interleaved, int dt,
                          void* stream) {
  if (!k || !steps || (!q) != (!q_out) || (!k_cache) != (!v_cache) || (!k_scales) != (!v_scales)) return TX_EINVAL;
  if ((!k_out && !k_cache) || (k_scales && !k_cache)) return TX_EINVAL;
  if (!(amplitude > 0.f) || !(amplitude < 3.0e38f)) return TX_EINVAL;
  if (norm != TX_NORM_NONE && norm != TX_NORM_RMS && norm != TX_NORM_LAYER) return TX_EINVAL;
  if (norm != TX_NORM_NONE && (!(eps >= 0.f) || !(eps < 3.0e38f))) return TX_EINVAL;
  if (norm != TX_NORM_LAYER && (q_bias || k_bias)) return TX_EINVAL;
  if (norm == TX_NORM_NONE && (q_weight || k_weight)) return TX_EINVAL;
  if (!q && (q_weight || q_bias)) return TX_EINVAL;
  int rc = check_seqs(tokens, batch, q_heads, kv_heads, head_dim, dt, cu_seqlens);
  if (rc != TX_OK) return rc;
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > head_dim) return TX_EINVAL;
  if (head_dim % 8 || head_dim > 256 || (k_scales && head_dim % 32)) return TX_EUNSUPPORTED;
  const void* params[4] = {q_weight, q_bias, k_weight, k_bias};
  bool any_param = false;
  for (const void* p : params) {
    any_param |= p != nullptr;
    if (!aligned16(p)) return TX_EUNSUPPORTED;
  }
  if (any_param && param_dt != dt && param_dt != TX_F32) return TX_EUNSUPPORTED;
  // (axes may share one row of positions, but not parts of rows)
  if (axes <= 0 || (positions && axes > 1 && positions_ld != 0 && positions_ld < tokens)) return TX_EINVAL;
  if (axes > 1 << 16 || positions_ld < 0 || positions_ld > (int64_t)1 << 40) return TX_EUNSUPPORTED;
  if (((uintptr_t)steps & 7u) || ((uintptr_t)positions & 7u) || ((uintptr_t)kv_lens & 3u) || ((uintptr_t)pair_axis & 3u))
    return TX_EUNSUPPORTED;
  // Without pair_axis every pair goes by axis 0; without positions there is one axis, the key index.
  if (!pair_axis || !positions) axes = 1;
  // Rows of one workgroup's tokens are counted in 32 bits.
  if ((q_heads + 2 * kv_heads) * head_dim > (int64_t)1 << 26) return TX_EUNSUPPORTED;
  if (q && (rc = check_rows(q, q_strides, tokens, q_heads, head_dim, false)) != TX_OK) return rc;
  if (q && (rc = check_rows(q_out, q_out_strides, tokens, q_heads, head_dim, true)) != TX_OK) return rc;
  if ((rc = check_rows(k, k_strides, tokens, kv_heads, head_dim, false)) != TX_OK) return rc;
  if (k_out && (rc = check_rows(k_out, k_out_strides, tokens, kv_heads, head_dim, true)) != TX_OK) return rc;
  const int size = k_scales ? 1 : 2;
  const int64_t blocks = head_dim / 32;
  if (k_cache) {
    if (!kv_lens) return TX_EINVAL;
    if ((rc = check_rows(v, v_strides, tokens, kv_heads, head_dim, false)) != TX_OK) return rc;
    if ((rc = check_pages(block_table, table_ld, batch, num_pages, page_size, max_pages)) != TX_OK) return rc;
    if ((rc = check_cache(k_cache, k_cache_strides, num_pages, kv_heads, page_size, head_dim, size)) != TX_OK) return rc;
    if ((rc = check_cache(v_cache, v_cache_strides, num_pages, kv_heads, page_size, head_dim, size)) != TX_OK) return rc;
    if (k_scales) {
      if ((rc = check_scales(k_scales, k_scales_strides, num_pages, kv_heads, page_size, blocks, 1)) != TX_OK) return rc;
      if ((rc = check_scales(v_scales, v_scales_strides, num_pages, kv_heads, page_size, blocks, 1)) != TX_OK) return rc;
    }
  }
  // Outputs: an input itself, or memory that no input and no other output uses.
  const int64_t param_bytes = (per_head ? q_heads : 1) * head_dim * (param_dt == TX_F32 ? 4 : 2);
  const int64_t k_param_bytes = (per_head ? kv_heads : 1) * head_dim * (param_dt == TX_F32 ? 4 : 2);
  const Mem none{};
  const Mem in[] = {mem_rows(k, k_strides, tokens, kv_heads, head_dim),
                    q ? mem_rows(q, q_strides, tokens, q_heads, head_dim) : none,
                    k_cache ? mem_rows(v, v_strides, tokens, kv_heads, head_dim) : none,
                    mem_span(q_weight, param_bytes), mem_span(q_bias, param_bytes), mem_span(k_weight, k_param_bytes),
                    mem_span(k_bias, k_param_bytes), mem_span(steps, rotary_dim / 2 * 8),
                    mem_span(pair_axis, rotary_dim / 2 * 4), mem_span(positions, ((axes - 1) * positions_ld + tokens) * 8),
                    mem_span(cu_seqlens, (batch + 1) * 4), mem_span(kv_lens, batch * 4),
                    k_cache ? mem_span(block_table, ((batch - 1) * table_ld + max_pages) * 4) : none};
  const Mem out[] = {k_out ? mem_rows(k_out, k_out_strides, tokens, kv_heads, head_dim) : none,
                     q ? mem_rows(q_out, q_out_strides, tokens, q_heads, head_dim) : none,
                     k_cache ? mem_pages(k_cache, k_cache_strides, num_pages, kv_heads, page_size, head_dim, size) : none,
                     k_cache ? mem_pages(v_cache, v_cache_strides, num_pages, kv_heads, page_size, head_dim, size) : none,
                     k_scales ? mem_pages(k_scales, k_scales_strides, num_pages, kv_heads, page_size, blocks, 1) : none,
                     k_scales ? mem_pages(v_scales, v_scales_strides, num_pages, kv_heads, page_size, blocks, 1) : none};
  for (int i = 0; i < (int)(sizeof(out) / sizeof(out[0])); ++i) {
    for (int j = 0; j < (int)(sizeof(in) / sizeof(in[0])); ++j) {
      if (i == 0 && j == 0 && k_out && same_rows(k_out, k_out_strides, k, k_strides)) continue;
      if (i == 1 && j == 1 && q && same_rows(q_out, q_out_strides, q, q_strides)) continue;
      if (!disjoint(out[i], in[j])) return TX_EINVAL;
    }
    for (int j = 0; j < i; ++j)
      if (!disjoint(out[i], out[j])) return TX_EINVAL;
  }
  NormRotaryArgs a{};
  a.s = {cu_seqlens, kv_lens, block_table, table_ld, (int)tokens, (int)batch, 0, 0, 0};
  a.k = k;
  a.k_st = k_strides[0];
  a.k_sh = k_strides[1];
  if (q) {
    a.q = q;
    a.q_st = q_strides[0];
    a.q_sh = q_strides[1];
    a.q_out = q_out;
    a.qo_st = q_out_strides[0];
    a.qo_sh = q_out_strides[1];
  }
  if (k_out) {
    a.k_out = k_out;
    a.ko_st = k_out_strides[0];
    a.ko_sh = k_out_strides[1];
  }
  if (k_cache) {
    a.s.num_pages = (int)num_pages;
    a.s.page_log2 = page_log2(page_size);
    a.s.max_pages = (int)max_pages;
    a.v = v;
    a.v_st = v_strides[0];
    a.v_sh = v_strides[1];
    a.k_cache = k_cache;
    a.kc_sp = k_cache_strides[0];
    a.kc_sh = k_cache_strides[1];
    a.kc_st = k_cache_strides[2];
    a.v_cache = v_cache;
    a.vc_sp = v_cache_strides[0];
    a.vc_sh = v_cache_strides[1];
    a.vc_st = v_cache_strides[2];
  }
  if (k_scales) {
    a.k_scales = k_scales;
    a.ks_sp = k_scales_strides[0];
    a.ks_sh = k_scales_strides[1];
    a.ks_st = k_scales_strides[2];
    a.v_scales = v_scales;
    a.vs_sp = v_scales_strides[0];
    a.vs_sh = v_scales_strides[1];
    a.vs_st = v_scales_strides[2];
  }
  a.q_weight = q_weight;
  a.q_bias = q_bias;
  a.k_weight = k_weight;
  a.k_bias = k_bias;
  a.param_f32 = param_dt == TX_F32 ? 1 : 0;
  a.param_sh = per_head ? (int)head_dim : 0;
  a.norm = norm;
  a.eps = eps;
  a.steps = (const uint64_t*)steps;
  a.pair_axis = pair_axis;
  a.positions = positions;
  a.positions_ld = positions_ld;
  a.axes = (int)axes;
  a.heads = (int)q_heads;
  a.kv_heads = (int)kv_heads;
  a.head_dim = (int)head_dim;
  a.rotary = (int)rotary_dim;
  a.amplitude = amplitude;
  a.interleaved = interleaved ? 1 : 0;
  return launch_norm_rotary_append(a, dt, (hipStream_t)stream);
}

int tx_cache_accept(void* k_cache, const int64_t k_cache_strides[3], uint8_t* k_scales,
                    const int64_t k_scales_strides[3], void* v_cache, const int64_t v_cache_strides[3],
                    uint8_t* v_scales, const int64_t v_scales_strides[3], const int32_t* cu_seqlens,
                    const int32_t* kv_lens, const int32_t* block_table, int64_t table_ld, const int32_t* path,
                    int64_t path_ld, int64_t max_path, const int32_t* counts, int32_t* lens_out, int64_t batch,
                    int64_t kv_heads, int64_t head_dim, int64_t num_pages, int64_t page_size, int64_t max_pages,
                    int dt, void* stream) {
  if (!k_cache || !v_cache || (!k_scales) != (!v_scales) || !kv_lens || !path || !counts || !lens_out) return TX_EINVAL;
  int rc = check_seqs(1, batch, kv_heads, kv_heads, head_dim, dt, cu_seqlens);
  if (rc != TX_OK) return rc;
  if (max_path <= 0 || path_ld < 0 || (batch > 1 && path_ld < max_path)) return TX_EINVAL;
  if (max_path > 1 << 24 || path_ld > (int64_t)1 << 40) return TX_EUNSUPPORTED;
  if (((uintptr_t)kv_lens & 3u) || ((uintptr_t)path & 3u) || ((uintptr_t)counts & 3u) || ((uintptr_t)lens_out & 3u))
    return TX_EUNSUPPORTED;
  if (head_dim % 8 || head_dim > 256 || (k_scales && head_dim % 32)) return TX_EUNSUPPORTED;
  if ((rc = check_pages(block_table, table_ld, batch, num_pages, page_size, max_pages)) != TX_OK) return rc;
  const int size = k_scales ? 1 : 2;
  const int64_t blocks = head_dim / 32;
  if ((rc = check_cache(k_cache, k_cache_strides, num_pages, kv_heads, page_size, head_dim, size)) != TX_OK) return rc;
  if ((rc = check_cache(v_cache, v_cache_strides, num_pages, kv_heads, page_size, head_dim, size)) != TX_OK) return rc;
  if (k_scales) {
    if ((rc = check_scales(k_scales, k_scales_strides, num_pages, kv_heads, page_size, blocks, 1)) != TX_OK) return rc;
    if ((rc = check_scales(v_scales, v_scales_strides, num_pages, kv_heads, page_size, blocks, 1)) != TX_OK) return rc;
  }
  // (lens_out is written while other workgroups of the sequence read kv_lens)
  const Mem none{};
  const Mem in[] = {mem_span(cu_seqlens, (batch + 1) * 4), mem_span(kv_lens, batch * 4), mem_span(counts, batch * 4),
                    mem_span(path, ((batch - 1) * path_ld + max_path) * 4),
                    mem_span(block_table, ((batch - 1) * table_ld + max_pages) * 4)};
  const Mem out[] = {mem_span(lens_out, batch * 4),
                     mem_pages(k_cache, k_cache_strides, num_pages, kv_heads, page_size, head_dim, size),
                     mem_pages(v_cache, v_cache_strides, num_pages, kv_heads, page_size, head_dim, size),
                     k_scales ? mem_pages(k_scales, k_scales_strides, num_pages, kv_heads, page_size, blocks, 1) : none,
                     k_scales ? mem_pages(v_scales, v_scales_strides, num_pages, kv_heads, page_size, blocks, 1) : none};
  for (int i = 0; i < 5; ++i) {
    for (const Mem& m : in)
      if (!disjoint(out[i], m)) return TX_EINVAL;
    for (int j = 0; j < i; ++j)
      if (!disjoint(out[i], out[j])) return TX_EINVAL;
  }
  CacheAcceptArgs a{};
  a.s = {cu_seqlens, kv_lens, block_table, table_ld, 0, (int)batch, (int)num_pages, page_log2(page_size), (int)max_pages};
  a.k_cache = k_cache;
  a.v_cache = v_cache;
  a.kc_sp = k_cache_strides[0] * size;
  a.kc_sh = k_cache_strides[1] * size;
  a.kc_st = k_cache_strides[2] * size;
  a.vc_sp = v_cache_strides[0] * size;
  a.vc_sh = v_cache_strides[1] * size;
  a.vc_st = v_cache_strides[2] * size;
  if (k_scales) {
    a.k_scales = k_scales;
    a.ks_sp = k_scales_strides[0];
    a.ks_sh = k_scales_strides[1];
    a.ks_st = k_scales_strides[2];
    a.v_scales = v_scales;
    a.vs_sp = v_scales_strides[0];
    a.vs_sh = v_scales_strides[1];
    a.vs_st = v_scales_strides[2];
  }
  a.path = path;
  a.path_ld = path_ld;
  a.counts = counts;
  a.lens_out = lens_out;
  a.max_path = (int)max_path;
  a.heads = (int)kv_heads;
  a.chunks = (int)(head_dim * size / 16);
  a.blocks = (int)blocks;
  return launch_cache_accept(a, (hipStream_t)stream);
}

}  // extern "C"
