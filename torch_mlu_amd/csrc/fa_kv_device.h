// Device-side helpers of the paged 8-bit cache's kernels (gfx950 only).
#ifndef FA_KV_DEVICE_H_
#define FA_KV_DEVICE_H_

#include "fa_device.h"
#include "fa_kv.h"

namespace fa {

typedef const __attribute__((address_space(4))) float* ConstF32Ptr;

// Stored bytes -> pairs of T.  Both formats have at most 8 significant bits and an exponent range that bf16 and fp16 hold, so
// the values are exact; e4m3's NaN stays NaN.
template <typename T, int F>
struct Stored;
template <>
struct Stored<__bf16, FA_KV_E4M3> {
  // bytes (0, 1) of w, or (2, 3)
  template <int HI>
  static __device__ __forceinline__ unsigned pair(unsigned w) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  }
};
template <>
struct Stored<_Float16, FA_KV_E4M3> {
  template <int HI>
  static __device__ __forceinline__ unsigned pair(unsigned w) {
    return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  }
};
template <typename T>
struct Stored<T, FA_KV_INT8> {
  template <int HI>
  static __device__ __forceinline__ unsigned pair(unsigned w) {
    return Mma<T>::pack2((float)(int8_t)(w >> (16 * HI)), (float)(int8_t)(w >> (16 * HI + 8)));
  }
};

// sequence b's query rows: first row and how many, clipped to what exists and to the longest the caller named
struct QRows {
  int first, count, aligned;  // aligned: the true length, which the causal mask goes by
  int64_t place;              // of its first row among those of all sequences
};
__device__ __forceinline__ QRows query_rows(const int32_t* cu, int b, int seqlen_q, int total_q) {
  if (!cu) return QRows{0, seqlen_q, seqlen_q, (int64_t)b * seqlen_q};
  const int first = min(max(cu[b], 0), total_q);
  const int n = min(max(cu[b + 1], first), total_q) - first;
  return QRows{first, min(n, seqlen_q), n, first};
}

}  // namespace fa

#endif  // FA_KV_DEVICE_H_
