/*
 * fa_rope.h — C ABI of rotary positions with one or several axes for MI355X (gfx950).  Exported by libfa_kv.so; the rules are
 * those of fa_fwd.h.  No counterpart in the reference.
 */
#ifndef FA_ROPE_H_
#define FA_ROPE_H_

#include "fa_fwd.h"

#ifdef __cplusplus
extern "C" {
#endif

#define FA_DTYPE_FP32 2 /* beside FA_DTYPE_FP16 and FA_DTYPE_BF16 */

#define FA_ROPE_MAX_AXES 8

/*
 * Each head's first 2 * pairs elements are turned, pair i by the angle positions[axes[i]][token] * inv_freq[i]:
 *   (a, b) -> (a cos - b sin, b cos + a sin)         (inverse: by the opposite angle, which is the gradient's way)
 * pair i is elements (i, i + pairs), or (2 i, 2 i + 1) when interleaved; elements from 2 * pairs on are copied.  Angles are
 * formed and reduced in 64 bits, products and sums are fp32, rounded once.  A token is (b, s) with b < batch, s < seqlen; its
 * head h of q lies at q + b q_stride_b + s q_stride_s + h q_stride_h.  q, k and their outputs may be the same memory with the
 * same strides (in place), and otherwise do not overlap.  heads_k = 0: no k.  An axis outside 0 ... num_axes - 1 counts as the
 * nearest one.
 */
typedef struct fa_rope_params {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  const void* positions; /* int32 or int64: axis a of token (b, s) at a pos_stride_a + b pos_stride_b + s pos_stride_s */
  const void* inv_freq;  /* [pairs] fp32 or fp64 */
  const int32_t* axes;   /* [pairs] */
  int64_t q_stride_b, q_stride_s, q_stride_h; /* elements */
  int64_t k_stride_b, k_stride_s, k_stride_h;
  int64_t qo_stride_b, qo_stride_s, qo_stride_h;
  int64_t ko_stride_b, ko_stride_s, ko_stride_h;
  int64_t pos_stride_a, pos_stride_b, pos_stride_s;
  int32_t batch, seqlen; /* >= 0 */
  int32_t heads_q;       /* > 0 */
  int32_t heads_k;       /* >= 0 */
  int32_t head_dim;      /* 2 ... 512 */
  int32_t pairs;         /* 1 ... head_dim / 2 */
  int32_t num_axes;      /* 1 ... FA_ROPE_MAX_AXES */
  int32_t dtype;         /* FA_DTYPE_* */
  int32_t positions_64;  /* 0: int32, 1: int64 */
  int32_t inv_freq_64;   /* 0: fp32, 1: fp64 */
  int32_t interleaved;   /* 0 / 1 */
  int32_t inverse;       /* 0 / 1 */
} fa_rope_params;

FA_API int fa_rope_validate(const fa_rope_params* p);
FA_API int fa_rope_launch(const fa_rope_params* p, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* FA_ROPE_H_ */
