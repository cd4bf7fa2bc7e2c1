// Host-only half of the launchers of include/fa_kv.h and include/fa_rope.h: argument validation, kernel choice and workspace
// sizes.  Plain C++ without any HIP construct, so that a CPU build with sanitizers can exercise it.
#ifndef FA_KV_HOST_H_
#define FA_KV_HOST_H_

#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include "fa_kv.h"
#include "fa_rope.h"

namespace fa {
namespace kvhost {

constexpr int64_t kMaxRowStride = 1 << 25;  // bytes between the rows of a page: 32 rows stay below a 32-bit offset

inline bool misaligned(const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) != 0; }
// n strides that are not negative and multiples of `unit`
inline bool bad_strides(const int64_t* s, int n, int64_t unit) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % unit) return true;
  return false;
}

inline int plan_validate(const fa_kv_plan_params* p) {
  if (!p) return FA_ERR_BAD_ARG;
  if (p->reserved != 0 || p->batch < 0 || p->table_pages < 0 || p->page_size <= 0 || p->max_tokens < 0 || p->free_capacity < 0) return FA_ERR_BAD_ARG;
  if (p->block_table_stride < p->table_pages) return FA_ERR_BAD_ARG;
  if (p->batch > FA_KV_MAX_BATCH) return FA_ERR_UNSUPPORTED;
  if ((int64_t)p->table_pages * p->page_size > 0x7fffffffLL) return FA_ERR_UNSUPPORTED;
  if (!p->free_count || !p->cu_seqlens || !p->free_left || p->free_count == p->free_left) return FA_ERR_BAD_ARG;
  if (p->batch > 0 && (!p->cached || !p->new_tokens || !p->seqused || !p->admitted || (!p->block_table && p->table_pages > 0))) return FA_ERR_BAD_ARG;
  if (p->max_tokens > 0 && (!p->positions || !p->slots)) return FA_ERR_BAD_ARG;
  if (p->free_capacity > 0 && !p->free_pages) return FA_ERR_BAD_ARG;
  const void* words[] = {p->cached, p->new_tokens, p->block_table, p->free_pages, p->free_count, p->cu_seqlens, p->seqused, p->positions, p->free_left};
  for (const void* w : words)
    if (misaligned(w, 4)) return FA_ERR_BAD_ARG;
  if (misaligned(p->slots, 8)) return FA_ERR_BAD_ARG;
  return FA_OK;
}

// what write and attention ask of a pool alike
template <typename P>
inline int pool_validate(const P* p) {
  const void* rows[] = {p->key_pages, p->value_pages};
  for (const void* r : rows)
    if (!r || misaligned(r, 16)) return FA_ERR_BAD_ARG;
  if (!p->key_scales || !p->value_scales || misaligned(p->key_scales, 4) || misaligned(p->value_scales, 4)) return FA_ERR_BAD_ARG;
  const int64_t bytes[] = {p->kp_stride_p, p->kp_stride_s, p->kp_stride_h, p->vp_stride_p, p->vp_stride_s, p->vp_stride_h};
  const int64_t scales[] = {p->ks_stride_p, p->ks_stride_b, p->ks_stride_h, p->vs_stride_p, p->vs_stride_b, p->vs_stride_h};
  if (bad_strides(bytes, 6, 16) || bad_strides(scales, 6, 1)) return FA_ERR_BAD_ARG;
  if (p->num_pages <= 0 || p->page_size <= 0 || p->scale_block <= 0 || p->head_dim <= 0) return FA_ERR_BAD_ARG;
  if (p->scale_block % 32 || p->page_size % p->scale_block || p->page_size > (1 << 20)) return FA_ERR_UNSUPPORTED;
  if (p->head_dim > 256 || p->head_dim % 16) return FA_ERR_UNSUPPORTED;
  if (p->dtype != FA_DTYPE_FP16 && p->dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED;
  if (p->format != FA_KV_E4M3 && p->format != FA_KV_INT8) return FA_ERR_UNSUPPORTED;
  if (p->kp_stride_s > kMaxRowStride || p->vp_stride_s > kMaxRowStride) return FA_ERR_UNSUPPORTED;
  if (p->kp_stride_p > 0x7fffffffLL || p->vp_stride_p > 0x7fffffffLL) return FA_ERR_UNSUPPORTED;
  for (int i = 0; i < 6; ++i)
    if (scales[i] > 0x7fffffffLL) return FA_ERR_UNSUPPORTED;
  return FA_OK;
}

inline int write_validate(const fa_kv_write_params* p) {
  if (!p) return FA_ERR_BAD_ARG;
  if (p->tokens < 0 || p->heads <= 0) return FA_ERR_BAD_ARG;
  if (const int rc = pool_validate(p)) return rc;
  if ((int64_t)p->num_pages * p->page_size > 0x7fffffffLL) return FA_ERR_UNSUPPORTED;
  if (p->heads > 65535) return FA_ERR_UNSUPPORTED;
  if (p->tokens > 0 && (!p->key || !p->value || !p->slots)) return FA_ERR_BAD_ARG;
  if (misaligned(p->key, 16) || misaligned(p->value, 16) || misaligned(p->slots, 8)) return FA_ERR_BAD_ARG;
  const int64_t st[] = {p->key_stride_t, p->key_stride_h, p->value_stride_t, p->value_stride_h};
  if (bad_strides(st, 4, 8)) return FA_ERR_BAD_ARG;
  return FA_OK;
}

inline int attn_validate(const fa_kv_attn_params* p) {
  if (!p) return FA_ERR_BAD_ARG;
  if (!p->q || !p->out || !p->lse || !p->block_table || !p->seqused_k) return FA_ERR_BAD_ARG;
  if (p->batch <= 0 || p->heads_q <= 0 || p->heads_k <= 0 || p->seqlen_q < 0 || p->table_pages < 0 || p->reserved != 0) return FA_ERR_BAD_ARG;
  if (p->cu_seqlens_q && p->total_q < 0) return FA_ERR_BAD_ARG;
  if (p->block_table_stride < p->table_pages) return FA_ERR_BAD_ARG;
  if (p->is_causal != FA_MASK_NONE && p->is_causal != FA_MASK_CAUSAL_BOTTOM_RIGHT) return FA_ERR_BAD_ARG;
  if (p->num_splits < 0 || p->num_splits > FA_MAX_SPLITS) return FA_ERR_BAD_ARG;
  if (const int rc = pool_validate(p)) return rc;
  if (p->heads_q % p->heads_k) return FA_ERR_UNSUPPORTED;
  if ((int64_t)p->table_pages * p->page_size > (1 << 29) || p->seqlen_q > (1 << 29)) return FA_ERR_UNSUPPORTED;
  if ((int64_t)p->seqlen_q * (p->heads_q / p->heads_k) > (1 << 30) || (int64_t)p->batch * p->heads_q > (1 << 30)) return FA_ERR_UNSUPPORTED;
  if (misaligned(p->q, 16) || misaligned(p->out, 16) || misaligned(p->lse, 4) || misaligned(p->block_table, 4) || misaligned(p->seqused_k, 4) ||
      misaligned(p->cu_seqlens_q, 4))
    return FA_ERR_BAD_ARG;
  const int64_t st[] = {p->q_stride_s, p->q_stride_h, p->o_stride_s, p->o_stride_h};
  const int64_t sb[] = {p->q_stride_b, p->o_stride_b};
  const int64_t sl[] = {p->lse_stride_h, p->lse_stride_s, p->cu_seqlens_q ? 0 : p->lse_stride_b};
  if (bad_strides(st, 4, 8) || (!p->cu_seqlens_q && bad_strides(sb, 2, 8)) || bad_strides(sl, 3, 1)) return FA_ERR_BAD_ARG;
  return FA_OK;
}

// How the call is cut: 16 * tiles (query row, head of the group) pairs a workgroup, `splits` slices of the key range.
struct AttnPlan {
  int32_t tiles;      // 1, 2 or 4 tiles of 16 rows: the streaming kernel; 8: the tile kernel
  int32_t row_blocks; // workgroups that share a (sequence, kv head, slice); packed, tile kernel: those of all sequences
  int32_t splits;
};
// Slices of the tile kernel: two workgroups share a CU (one at head_dim 256), and one that has it to itself takes two thirds of
// the time; a start and an end cost about 5 tiles, the join of the slices 2 and its partial results' bytes, of which 11 MB pass
// while a tile is computed.  Measured (us, bf16, 32 / 8 heads, head_dim 128, e4m3; in the chosen number of slices, in one, in the
// nearest others): 500 rows over 32768 keys 324 in 4 (829; 399 in 3, 344 in 6), 4 x 512 over 4096 168 in 1 (178 in 2), packed
// prompts and decodes 16 x 512 over 4096 198 in 2 (206; 201 in 3), 4 x 512 over 16384 212 in 3 (423; 298 in 2, 232 in 4).
inline int64_t tile_slices(int64_t units, int64_t tiles, int64_t rows, int head_dim) {
  const double slots = head_dim > 128 ? 256 : 512;
  double least = 0;
  int64_t best = 1;
  for (int64_t n = 1; n <= FA_MAX_SPLITS && (n == 1 || tiles >= 8 * n); ++n) {
    const double x = (double)units * (double)n / slots, whole = floor(x), part = x - whole;
    const double rounds = whole + (part == 0 ? 0 : (part <= 0.5 ? 0.66 : 1));
    const double cost = rounds * ((double)tiles / (double)n + 5) + (n > 1 ? 2 + (double)rows * (double)n * (8.0 * head_dim + 16) / 11e6 : 0);
    if (n == 1 || cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

// query rows of all sequences, those that no packed sequence owns among them
inline int64_t attn_rows(const fa_kv_attn_params* p) { return p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q; }
inline AttnPlan attn_plan(const fa_kv_attn_params* p) {
  AttnPlan r;
  const int64_t rows = (int64_t)p->seqlen_q * (p->heads_q / p->heads_k);
  r.tiles = rows <= 16 ? 1 : (rows <= 32 ? 2 : (rows <= 64 && p->head_dim <= 128 ? 4 : 8));
  r.row_blocks = (int32_t)((rows + 16 * r.tiles - 1) / (16 * r.tiles));
  if (r.row_blocks < 1) r.row_blocks = 1;
  const int64_t keys = (int64_t)p->table_pages * p->page_size;
  const int64_t blocks = r.tiles == 8 ? (keys + 63) / 64 : (keys + 31) / 32;
  int64_t units = (int64_t)p->batch * p->heads_k * r.row_blocks;
  if (r.tiles == 8 && p->cu_seqlens_q) {
    // a sequence with c rows before it begins at place c * group / 128 + its number
    const int64_t places = (int64_t)p->total_q * (p->heads_q / p->heads_k) / 128 + p->batch;
    r.row_blocks = places > 0x7fffffff ? 0x7fffffff : (int32_t)places;
    units = places * p->heads_k;
  }
  int64_t n = p->num_splits;
  if (n == 0) {
    n = 1;
    if (r.tiles == 8) {
      n = tile_slices(units, blocks, attn_rows(p) * p->heads_q, p->head_dim);
    } else {
      while (n * 2 <= FA_MAX_SPLITS && units * n * 2 <= 1024 && keys / (n * 2) >= 256) n *= 2;
    }
  }
  if (n > blocks) n = blocks > 0 ? blocks : 1;
  // partial sums within 1 GiB
  const int64_t slots = attn_rows(p) * p->heads_q;
  while (n > 1 && slots > (1LL << 30) / (n * (p->head_dim * 4 + 8))) n /= 2;
  r.splits = (int32_t)n;
  return r;
}
inline size_t attn_workspace_bytes(const fa_kv_attn_params* p, const AttnPlan& r) {
  if (r.splits <= 1) return 0;
  return (size_t)attn_rows(p) * p->heads_q * r.splits * ((size_t)p->head_dim * 4 + 8);
}

inline int rope_validate(const fa_rope_params* p) {
  if (!p) return FA_ERR_BAD_ARG;
  if (p->batch < 0 || p->seqlen < 0 || p->heads_q <= 0 || p->heads_k < 0 || p->head_dim < 2 || p->pairs < 1 || p->pairs > p->head_dim / 2) return FA_ERR_BAD_ARG;
  if (p->num_axes < 1 || ((p->positions_64 | p->inv_freq_64 | p->interleaved | p->inverse) & ~1)) return FA_ERR_BAD_ARG;
  if (p->dtype != FA_DTYPE_FP16 && p->dtype != FA_DTYPE_BF16 && p->dtype != FA_DTYPE_FP32) return FA_ERR_UNSUPPORTED;
  if (p->head_dim > 512 || p->num_axes > FA_ROPE_MAX_AXES || p->heads_q > (1 << 20) || p->heads_k > (1 << 20)) return FA_ERR_UNSUPPORTED;
  if ((int64_t)p->batch * p->seqlen > 0x7fffffffLL) return FA_ERR_UNSUPPORTED;
  if (!p->inv_freq || !p->axes || misaligned(p->axes, 4) || misaligned(p->inv_freq, p->inv_freq_64 ? 8 : 4)) return FA_ERR_BAD_ARG;
  const uintptr_t size = p->dtype == FA_DTYPE_FP32 ? 4 : 2;
  if ((int64_t)p->batch * p->seqlen > 0) {
    if (!p->q || !p->q_out || !p->positions || (p->heads_k > 0 && (!p->k || !p->k_out))) return FA_ERR_BAD_ARG;
    if (misaligned(p->q, size) || misaligned(p->q_out, size) || misaligned(p->positions, p->positions_64 ? 8 : 4)) return FA_ERR_BAD_ARG;
    if (p->heads_k > 0 && (misaligned(p->k, size) || misaligned(p->k_out, size))) return FA_ERR_BAD_ARG;
  }
  return FA_OK;
}
// 16-byte pieces of a head: where every row starts at one and a piece has the pairs of one side, or whole pairs
inline bool rope_vector(const fa_rope_params* p) {
  const int64_t n = p->dtype == FA_DTYPE_FP32 ? 4 : 8;
  if (p->head_dim % n || (p->interleaved ? (2 * p->pairs) % n : p->pairs % n)) return false;
  if (misaligned(p->q, 16) || misaligned(p->q_out, 16)) return false;
  int64_t all = p->q_stride_b | p->q_stride_s | p->q_stride_h | p->qo_stride_b | p->qo_stride_s | p->qo_stride_h;
  if (p->heads_k > 0) {
    if (misaligned(p->k, 16) || misaligned(p->k_out, 16)) return false;
    all |= p->k_stride_b | p->k_stride_s | p->k_stride_h | p->ko_stride_b | p->ko_stride_s | p->ko_stride_h;
  }
  return (all & (n - 1)) == 0;
}

}  // namespace kvhost
}  // namespace fa

#endif  // FA_KV_HOST_H_
