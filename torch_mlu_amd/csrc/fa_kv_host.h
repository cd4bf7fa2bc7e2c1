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

constexpr int64_t kMaxRowStride = (1 << 24) - 1;  // bytes between the rows of a page: an operand of a 24-bit product

// a launch's threads are counted in 32 bits
inline bool grid_fits(int64_t wgs, int64_t threads) { return wgs <= 0xffffffffLL / threads; }

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
  if (!p->free_count || !p->cu_seqlens || !p->free_left) return FA_ERR_BAD_ARG;
  if (p->batch > 0 && (!p->cached || !p->new_tokens || !p->seqused || !p->admitted || (!p->block_table && p->table_pages > 0))) return FA_ERR_BAD_ARG;
  if (p->max_tokens > 0 && (!p->positions || !p->slots)) return FA_ERR_BAD_ARG;
  if (p->free_capacity > 0 && !p->free_pages) return FA_ERR_BAD_ARG;
  const void* words[] = {p->cached, p->new_tokens, p->block_table, p->free_pages, p->free_count, p->cu_seqlens, p->seqused, p->positions, p->free_left};
  for (const void* w : words)
    if (misaligned(w, 4)) return FA_ERR_BAD_ARG;
  if (misaligned(p->slots, 8)) return FA_ERR_BAD_ARG;
  // workgroups read lengths and the count while others already write
  const void* in[] = {p->cached, p->new_tokens, p->free_count, p->free_pages, p->block_table};
  const void* out[] = {p->cu_seqlens, p->seqused, p->positions, p->slots, p->admitted, p->free_left};
  for (const void* i : in)
    for (const void* o : out)
      if (i && i == o) return FA_ERR_BAD_ARG;
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

// The write kernel: wavefronts that share a run of rows, the tokens whose runs they look for, workgroups of a call.
// A wavefront's registers hold kWriteLoads x 1 KiB of rows; four share a run where whole blocks are longer (us, one and four: 2 x
// 7143 rows of 16 heads of 96, blocks of 128 55 and 37; 3 x 4493 of 16 of 256, blocks of 64 69 and 49; 64 x 24 of 16 of 128,
// blocks of 256 9.7 and 12.5).  Looking through tokens that begin no run costs wavefronts, several runs for one cost time: as few
// tokens each as leave 4096 wavefronts (us, 32 tokens and this rule: 1024 x 1 of 8 heads of 128 50 and 19, 128 x 8 13.6 and 7.0,
// 8 x 2000 19 and 19, of 8 tokens 36).
constexpr int kWriteLoads = 16;
inline int write_waves(const fa_kv_write_params* p) {
  const int fits = kWriteLoads * (512 / p->head_dim);
  return p->scale_block > fits && p->tokens > fits ? 4 : 1;
}
inline int32_t write_chunk(const fa_kv_write_params* p) {
  int32_t n = 1;
  while (n < 32 && (int64_t)p->tokens * 2 * p->heads > (int64_t)n * 4096) n *= 2;
  return n;
}
inline int64_t write_wgs(const fa_kv_write_params* p) {
  const int64_t units = ((int64_t)p->tokens + write_chunk(p) - 1) / write_chunk(p) * 2 * p->heads, per_wg = 4 / write_waves(p);
  return (units + per_wg - 1) / per_wg;
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
  if (!grid_fits(write_wgs(p), 256)) return FA_ERR_UNSUPPORTED;
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

// How the call is cut: 16 * tiles (query row, head of the group) pairs a workgroup and head, `splits` slices of the key range.
struct AttnPlan {
  int32_t tiles;      // 1 or 2 tiles of 16 rows: the streaming kernel; 8: the tile kernel
  int32_t hw_log2;    // streaming kernel: log2 of the neighbouring kv heads of a workgroup
  int32_t row_blocks; // tile kernel: workgroups that share a (sequence, kv head, slice); packed: those of all sequences
  int32_t splits;
};
// wavefronts of the streaming kernel's workgroups: as many as a CU's registers hold once at least
constexpr int stream_waves(int dp) { return dp <= 128 ? 8 : 4; }
// query rows of all sequences, those that no packed sequence owns among them
inline int64_t attn_rows(const fa_kv_attn_params* p) { return p->cu_seqlens_q ? p->total_q : (int64_t)p->batch * p->seqlen_q; }

// Slices of the tile kernel: two workgroups share a CU (one at head_dim 256), and one that has it to itself takes two thirds of
// the time; a start and an end cost about 5 tiles, the join of the slices 2 and its partial results' bytes, of which 11 MB pass
// while a tile is computed.  Measured (us, bf16, 32 / 8 heads, head_dim 128, e4m3; in the chosen number of slices, in one, in the
// nearest others): 500 rows over 32768 keys 317 in 4 (845; 405 in 3, 340 in 6), 4 x 512 over 4096 168 in 1 (178 in 2), 4 x 512 over
// 16384 212 in 3 (423; 298 in 2, 232 in 4).  Packed batches of prompts and single tokens have lengths of all sizes, so that rounds
// run into one another: six tenths of their number, and half of a longest block at the end.  16 x 512 over 4096 176 in 1 (183 in 2),
// 64 x 256 over 2048 167 in 1 (203 in 2), 28 / 4 heads, 8 x 1024 over 8192 262 in 3 (261; 273 in 2), 16 / 4 heads, 40 x 300 over
// 6000 180 in 3 (190; 188 in 2, 171 in 4), 16 / 16 heads, 6 x 2000 over 4000 130 in 1 (143 in 2).
inline int64_t tile_slices(int64_t units, int64_t tiles, int64_t rows, int head_dim, bool packed) {
  const double slots = head_dim > 128 ? 256 : 512;
  double least = 0;
  int64_t best = 1;
  for (int64_t n = 1; n <= FA_MAX_SPLITS && (n == 1 || tiles >= 2 * n); ++n) {
    const double x = (double)units * (double)n / slots, whole = floor(x), part = x - whole;
    const double rounds = packed ? (x > 0.83 ? 0.6 * x + 0.5 : 1) : whole + (part == 0 ? 0 : (part <= 0.5 ? 0.66 : 1));
    const double cost = rounds * ((double)tiles / (double)n + 5) + (n > 1 ? (packed ? 8 : 2) + (double)rows * (double)n * (8.0 * head_dim + 16) / 11e6 : 0);
    if (n == 1 || cost < least) {
      least = cost;
      best = n;
    }
  }
  return best;
}

// Slices of the streaming kernel: workgroups for every CU while a slice keeps a block for each of its turns, and beyond 4096
// keys slices of 1024, which even out different lengths and a last round of long ones; of 4096 where every CU has a workgroup
// anyway, as a full batch has nothing to even out (64 x 8192, lengths 15/16 ... 1: 186 in 1, 191 in 2, 200 in 8).  Measured (us, e4m3, 32 / 8 heads,
// head_dim 128, lengths 1/4 ... 1 of the given; the chosen number of slices: time; others): 1 x 4097 32: 10.0; 16: 11.3,
// 64: 10.3.  4 x 8192 16: 16.5; 8: 20, 32: 17.  16 x 2048 4: 15.4; 2: 19.6, 8: 16.7.  64 x 2048 1: 34.4; 2: 35.5.  16 x 16384
// 16: 59; 4: 74, 8: 68, 32: 60.  64 x 8192 2: 149; 1: 153, 8: 142.  256 x 4096 1: 283; 2: 276.  28 / 4 heads, 128 x 4096
// 1: 73; 2: 76.  Two neighbouring heads a workgroup against one, four and eight, each in its best number of slices: 1 x 4097
// 10.0, 10.2, 10.4, 13.0; 64 x 8192 142, 147, 141, 141; 64 x 2048 34, 34, 37, 37; 256 x 4096 276, 291, 272, 277; 28 / 4 heads,
// int8, 32 x 5000, two rows 32, 31, 34.
inline int64_t stream_slices(int64_t units, int64_t turns, int64_t keys) {
  int64_t n = (256 + units - 1) / units;
  const int64_t most = keys / (32 * turns);
  if (n > most) n = most;
  if (n < 1) n = 1;
  const int64_t longest = units >= 256 ? 4096 : 1024;
  if (keys > 4096)
    while (n * 2 <= FA_MAX_SPLITS && keys > longest * n && units * n < 2048) n *= 2;
  return n < FA_MAX_SPLITS ? n : FA_MAX_SPLITS;
}

inline AttnPlan attn_plan(const fa_kv_attn_params* p) {
  AttnPlan r;
  const int64_t group = p->heads_q / p->heads_k, rows = (int64_t)p->seqlen_q * group;
  // (beyond 32 rows a conversion that serves one wavefront costs more than tiles that are shared: us, streaming with 4 tiles of
  // rows and tile kernel, 28 / 4 heads, 12 x 8 rows over 6757 keys 60 and 38, 32 / 8, 1 x 16 over 32768 50 and 41, 16 / 1, int8,
  // 64 x 4 over 8000 80 and 53; 17 ... 32 rows with 2 tiles, 32 / 8, 64 x 8 over 4096 85 and 117, 16 x 8 over 8192 57 and 66)
  r.tiles = rows <= 16 ? 1 : (rows <= 32 ? 2 : 8);
  r.row_blocks = 1;
  r.hw_log2 = 0;
  const int64_t keys = (int64_t)p->table_pages * p->page_size;
  const int64_t blocks = r.tiles == 8 ? (keys + 63) / 64 : (keys + 31) / 32;
  int64_t n = p->num_splits;
  if (r.tiles == 8) {
    // (packed: a sequence with c rows before it begins at place c * group / 128 + its number)
    const int64_t places = p->cu_seqlens_q ? (int64_t)p->total_q * group / 128 + p->batch : (rows + 127) / 128;
    r.row_blocks = places > 0x7fffffff ? 0x7fffffff : (int32_t)places;
    // (blocks of few rows count half: they fill the gaps that the others leave)
    const int64_t units = p->cu_seqlens_q ? (int64_t)p->total_q * group / 128 + p->batch / 2 : places * p->batch;
    if (n == 0) n = tile_slices((units > 0 ? units : 1) * p->heads_k, blocks, attn_rows(p) * p->heads_q, p->head_dim, p->cu_seqlens_q != nullptr);
  } else {
    const int dp = p->head_dim <= 64 ? 64 : (p->head_dim <= 128 ? 128 : 256), waves = stream_waves(dp);
    r.hw_log2 = p->heads_k % 2 == 0 ? 1 : 0;
    if (n == 0) n = stream_slices((int64_t)p->batch * (p->heads_k >> r.hw_log2), waves >> r.hw_log2, keys);
  }
  if (n > blocks) n = blocks > 0 ? blocks : 1;
  // partial sums within 1 GiB
  const int64_t slots = attn_rows(p) * p->heads_q;
  while (n > 1 && slots > (1LL << 30) / (n * (p->head_dim * 4 + 8))) n /= 2;
  r.splits = (int32_t)n;
  return r;
}
// workgroups of the call; below 0: more than a launch can have
inline int64_t attn_wgs(const fa_kv_attn_params* p, const AttnPlan& r) {
  if (r.tiles != 8) {
    const int64_t n = (int64_t)p->batch * (p->heads_k >> r.hw_log2) * r.splits;
    return grid_fits(n, 512) ? n : -1;
  }
  const int64_t per_row_block = p->cu_seqlens_q ? (int64_t)p->heads_k * r.splits : ((int64_t)p->batch * p->heads_k * r.splits + 7) / 8 * 8;
  return per_row_block <= 0xffffffffLL / 256 / r.row_blocks ? per_row_block * r.row_blocks : -1;
}
inline size_t attn_workspace_bytes(const fa_kv_attn_params* p, const AttnPlan& r) {
  if (r.splits <= 1) return 0;
  return (size_t)attn_rows(p) * p->heads_q * r.splits * ((size_t)p->head_dim * 4 + 8);
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
// Tokens of a workgroup: as many as give each of its threads two pieces, while the workgroups stay four a CU (us, one token and
// this rule: 16384 tokens of 2 + 1 heads of 64 16.3 and 6.2, of 8 + 8 of 128 28.3 and 23.4; 2000 of 32 + 8 of 128 9.5 and 9.4).
inline int32_t rope_tokens_per_wg(const fa_rope_params* p, bool vec) {
  const int64_t e = vec ? (p->dtype == FA_DTYPE_FP32 ? 4 : 8) : 1, tokens = (int64_t)p->batch * p->seqlen;
  const int64_t turned = (p->interleaved && vec ? 2 * p->pairs : p->pairs) / e, copied = (p->head_dim - 2 * p->pairs) / e;
  const int64_t pieces = (turned + copied) * ((int64_t)p->heads_q + p->heads_k);
  int32_t n = 1;
  while (n < 16 && n * 2 * pieces <= 512 && tokens / (n * 2) >= 1024) n *= 2;
  return n;
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
    const int64_t per_wg = rope_tokens_per_wg(p, rope_vector(p));
    if (!grid_fits(((int64_t)p->batch * p->seqlen + per_wg - 1) / per_wg, 256)) return FA_ERR_UNSUPPORTED;
  }
  return FA_OK;
}

}  // namespace kvhost
}  // namespace fa

#endif  // FA_KV_HOST_H_
