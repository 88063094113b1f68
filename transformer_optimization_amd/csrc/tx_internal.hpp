// Internal launcher interface between the C-ABI layer (api.hip) and the
// kernel translation units.  Arguments arrive here already validated.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "limits.hpp"
#include "tx_api.h"

namespace tx {

struct LayerNormArgs {
  const void* x;
  const void* delta;
  void* x_out;
  void* y;
  const void* gamma;
  const void* beta;
  const uint8_t* row_valid;
  float* mean_out;
  float* rstd_out;
  int64_t rows;
  int64_t d;
  float eps;
  int x_dt, y_dt, param_dt;
  uint32_t flags;
};

struct GemmArgs {
  const void* a;
  const void* w;
  const void* bias;
  const void* res;
  void* c;
  const uint8_t* row_valid;
  int64_t lda, ldw, ldr, ldc;
  int m, n, k;
  uint32_t epi;
  // Packed-QKV split store (tx_qkv_proj): columns >= qk_cols go to vt.
  void* vt;
  int64_t ldvt;
  int qk_cols;  // 2 * d_model
  int seq;
  int heads;
  int head_dim;
  int group;  // tile rows per band of the tile order (set by launch_gemm)
  // 1: 16-byte staged epilogue; 2 (gemm_hp_kernel only): V^T columns staged too.
  // Set by launch_hp and gemm_ring.hip's launch_cfg.
  int stage16;
};

// Attention operands as strided [batch, head, seq, head_dim] views (element
// strides sb / sh / ss; head_dim contiguous).  V is either natural
// (vnat = 1: v[b, h, s, d] = v + b*v_sb + h*v_sh + s*v_ss + d) or head-
// transposed (vnat = 0: v[b, h, s, d] = v + b*v_sb + h*v_sh + d*ldvt + s).
struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  int64_t q_sb, q_sh, q_ss;
  int64_t k_sb, k_sh, k_ss;
  int64_t v_sb, v_sh, v_ss;
  int64_t o_sb, o_sh, o_ss;
  const uint8_t* key_valid;  // key_valid[b * kv_sb + s]; nullptr = all valid
  int64_t kv_sb;
  int vnat;
  int64_t ldvt;              // vnat = 0: keys per transposed row
  int batch, seq, heads, head_dim;
  float scale;
  int causal;
  int softmax_mode;   // TX_SOFTMAX_EAGER or TX_SOFTMAX_ONLINE
  float* row_stats;   // eager mode: [B*H*S][2] (max, sum) workspace
};

// x / d for 0 <= x < 2^31 and a d that only the call knows: (mulhi(x, m) + x)
// >> s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1.
struct SeqDiv {
  uint32_t d, m, s;
};
inline SeqDiv seq_div_by(int d) {
  SeqDiv v{(uint32_t)d, 0, 0};
  while (((uint64_t)1 << v.s) < (uint64_t)d) ++v.s;
  v.m = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << v.s) - (uint64_t)d)) / (uint64_t)d + 1);
  return v;
}

// Packed sequences and a paged cache (tx_api.h).  Strides in elements: st per
// token (or slot), sh per head, sp per page.
struct SeqArgs {
  const int32_t* cu;        // [batch + 1]
  const int32_t* kv_lens;   // [batch] or nullptr (as many keys as rows)
  const int32_t* table;     // [batch][table_ld] page indices (paged only)
  int64_t table_ld;
  int tokens, batch;
  int num_pages, page_log2, max_pages;
};

struct RotaryArgs {
  SeqArgs s;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* k_cache;
  void* v_cache;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh;
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  const uint64_t* steps;
  const int64_t* positions;
  int heads, kv_heads, head_dim, rotary;
  float amplitude;
  int interleaved;
  // Work units (rotary.hip): of a head of q or k, of a token; and division by them.
  int turn_units, single_units, units;
  SeqDiv by_units, by_v_units, by_token;
};

// rotary_append with norms, positions of several axes and 8-bit caches.  Strides
// of caches and scales are in their own elements (a code or a scale: a byte).
struct NormRotaryArgs {
  SeqArgs s;
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* k_cache;
  void* v_cache;
  uint8_t* k_scales;  // nullptr: 16-bit caches
  uint8_t* v_scales;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh;
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  int64_t ks_sp, ks_sh, ks_st, vs_sp, vs_sh, vs_st;
  const void* q_weight;  // gains and shifts; each may be nullptr
  const void* q_bias;
  const void* k_weight;
  const void* k_bias;
  int param_f32;  // they are fp32 (else of the tensors' type)
  int param_sh;   // elements from one head's to the next's: head_dim, or 0
  int norm;       // TX_NORM_*
  float eps;
  const uint64_t* steps;
  const int32_t* pair_axis;
  const int64_t* positions;
  int64_t positions_ld;
  int axes;
  int heads, kv_heads, head_dim, rotary;
  float amplitude;
  int interleaved;
  SeqDiv by_heads, by_kv_heads, by_half;
};

struct CacheAcceptArgs {
  SeqArgs s;
  void* k_cache;
  void* v_cache;
  uint8_t* k_scales;  // nullptr: 16-bit caches
  uint8_t* v_scales;
  // bytes
  int64_t kc_sp, kc_sh, kc_st, vc_sp, vc_sh, vc_st;
  int64_t ks_sp, ks_sh, ks_st, vs_sp, vs_sh, vs_st;
  const int32_t* path;
  int64_t path_ld;
  const int32_t* counts;
  int32_t* lens_out;
  int max_path, heads;
  int chunks, blocks;  // 16-byte chunks and scales of a head's row
};

struct SeqAttnArgs {
  SeqArgs s;
  const void* q;
  const void* k;  // [T][kv_heads][hd], or the cache
  const void* v;
  void* o;
  int64_t q_st, q_sh, o_st, o_sh;
  int64_t k_sp, k_sh, k_st, v_sp, v_sh, v_st;
  int heads, kv_heads, group, head_dim;
  SeqDiv by_group, by_kv_heads;
  float scale;
  int causal;
  int paged;
  int64_t max_q_len;
  int few;   // rows of a tile where every sequence has few rows (seq_common.hpp), else 0
  int few_parts;  // most parts of the keys of such rows
  int call_items;  // of tiles, where the call's totals cut their keys, else 0
  int cus;
  float* ws;     // partial results: [rows][head_dim], normalised,
  float* ws_ml;  // and their maxima (log2 units) and sums, [rows][2]
  // 8-bit caches (strides of k and v in bytes): scales, one byte for 32 elements.
  const uint8_t* k_scales;  // nullptr: 16-bit caches
  const uint8_t* v_scales;
  int64_t ks_sp, ks_sh, ks_st, vs_sp, vs_sh, vs_st;
  // Draft trees: which of its sequence's new tokens a token sees.
  const uint64_t* tree;  // nullptr: none
  int64_t tree_ld;
  int tree_words;
};

int launch_rotary_append(const RotaryArgs& a, int dt, hipStream_t st);
int launch_seq_attention(const SeqAttnArgs& a, int dt, hipStream_t st);
int launch_norm_rotary_append(const NormRotaryArgs& a, int dt, hipStream_t st);
int launch_cache_accept(const CacheAcceptArgs& a, hipStream_t st);
// Paged attention over an 8-bit cache, or of a draft tree, or both.
int launch_cache_attention(const SeqAttnArgs& a, int dt, hipStream_t st);
// Floats of workspace a paged call of these sizes needs; over an 8-bit cache or of a draft tree.
int64_t seq_attention_workspace(const SeqAttnArgs& a);
int64_t cache_attention_workspace(const SeqAttnArgs& a);

int launch_layernorm(const LayerNormArgs& a, hipStream_t st);
int launch_gemm(const GemmArgs& g, int ab_dt, int c_dt, int bias_dt, int res_dt, bool qkv,
                hipStream_t st);
// gemm_ring.hip (K a multiple of 64, vector-aligned C, 32-bit tile offsets): the
// launch of tile configuration cfg (gemm_route.hpp).
int launch_gemm_ring(const GemmArgs& g, int ab_dt, int c_dt, int res_dt, bool qkv, int cfg, bool ks4,
                     hipStream_t st);
int launch_attention(const AttnArgs& a, int dt, hipStream_t st);
int device_cu_count();
// The variant of op (TX_SELECT_*) that this thread or the process's environment
// asks for; -1: the dispatcher's own choice.
int selected_kernel(int op);
// Shared memory per block of the current device, as the HIP runtime reports
// it to every library on the device (0 if it cannot be queried).
int64_t device_shared_mem_per_block();
// Device address of the current device's fixed attention scratch
// (2 * TX_NOALLOC_MAX_STAT_ROWS floats); nullptr if it cannot be resolved.
float* scratch_device_ptr();

}  // namespace tx
