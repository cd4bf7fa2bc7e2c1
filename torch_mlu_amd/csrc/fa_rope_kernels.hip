// Rotary positions with one or several axes: the kernels and the C ABI of fa_rope_* (include/fa_rope.h).
//
//   t = position[axis of the pair] * inv_freq[pair],   (a, b) -> (a cos t - b sin t, b cos t + a sin t)
//
// The gradient of the inputs is the outputs' gradient turned by -t, so the backward pass is the same kernel.
#include <hip/hip_runtime.h>

#include "fa_device.h"
#include "fa_kv_host.h"

namespace {
using namespace fa;

struct RArgs {
  const unsigned char* x[2];  // q, k
  unsigned char* y[2];
  const void* positions;
  const void* freq;
  const int32_t* axes;
  int64_t x_sb[2], x_ss[2], x_sh[2], y_sb[2], y_ss[2], y_sh[2];  // bytes
  int64_t pos_sa, pos_sb, pos_ss;                                // elements
  int32_t tokens, seqlen, heads[2], head_dim, pairs, num_axes;
  int32_t positions_64, freq_64, interleaved, inverse;
  int32_t per_wg;  // tokens of a workgroup
};

template <typename T>
struct Io;
template <>
struct Io<float> {
  static __device__ __forceinline__ float get(const unsigned char* p) { return *(const float*)p; }
  static __device__ __forceinline__ void put(unsigned char* p, float x) { *(float*)p = x; }
  static __device__ __forceinline__ void unpack(u32x4 w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __builtin_bit_cast(float, (unsigned)w[i]);
  }
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(unsigned, x[i]);
    return w;
  }
};
template <typename T>
struct Io {
  static __device__ __forceinline__ float get(const unsigned char* p) { return Mma<T>::to_float(*(const unsigned short*)p); }
  static __device__ __forceinline__ void put(unsigned char* p, float x) { *(T*)p = (T)x; }
  static __device__ __forceinline__ void unpack(u32x4 w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = Mma<T>::to_float((unsigned short)(w[i] & 0xffffu));
      x[2 * i + 1] = Mma<T>::to_float((unsigned short)(w[i] >> 16));
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float* x) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = Mma<T>::pack2(x[2 * i], x[2 * i + 1]);
    return w;
  }
};

// The angles of a token's pairs are the same for all its heads: a workgroup works them out once for its tokens, in LDS, and
// then only moves data.  An angle is formed in turns in 64 bits and its whole turns dropped there, so that it is as exact far
// into a long prompt as at its start (in 32 bits position 10^6 would be off by 0.06 rad); sine and cosine are 32 bits of that.
// Bound by memory: 16384 tokens of 16 + 16 heads, head_dim 128, bf16: 57 us, 4.7 TB/s read and written, of 4.95 that a copy reaches.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) fa_rope_kernel(const RArgs a) {
  extern __shared__ __attribute__((aligned(16))) float2 table[];  // [per_wg][pairs]: cos, sin
  const int tid = threadIdx.x, n = a.pairs, D = a.head_dim;
  const int64_t t0 = (int64_t)blockIdx.x * a.per_wg;
  const int tokens = (int)min((int64_t)a.per_wg, a.tokens - t0);
  for (int i = tid; i < tokens * n; i += 256) {
    const int tt = i / n, pr = i - tt * n;
    const int64_t t = t0 + tt;
    const int b = (int)(t / a.seqlen), s = (int)(t - (int64_t)b * a.seqlen);
    const int ax = min(max(a.axes[pr], 0), a.num_axes - 1);
    const int64_t at = ax * a.pos_sa + b * a.pos_sb + s * a.pos_ss;
    const double pos = a.positions_64 ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
    const double freq = a.freq_64 ? ((const double*)a.freq)[pr] : (double)((const float*)a.freq)[pr];
    const double turns = pos * (freq * 0.15915494309189535);
    const float half_turns = (float)(2.0 * (turns - rint(turns)));
    float sn, cs;
    sincospif(half_turns, &sn, &cs);
    table[i] = float2{cs, a.inverse ? -sn : sn};
  }
  __syncthreads();

  constexpr int E = VEC ? 16 / (int)sizeof(T) : 1;  // elements of a piece
  const int heads = a.heads[0] + a.heads[1];
  // pieces of a head: with the halves apart one has both sides of E pairs, interleaved E elements; then what is only copied
  const int turned = a.interleaved ? (VEC ? 2 * n / E : n) : n / E;
  const int copied = (D - 2 * n) / E, pieces = turned + copied;
  const int items = tokens * heads * pieces;
  for (int i = tid; i < items; i += 256) {
    const int th = i / pieces, pc = i - th * pieces;
    const int tt = th / heads, hh = th - tt * heads;
    const int64_t t = t0 + tt;
    const int b = (int)(t / a.seqlen), s = (int)(t - (int64_t)b * a.seqlen);
    const int which = hh >= a.heads[0] ? 1 : 0, h = hh - (which ? a.heads[0] : 0);
    const unsigned char* x = a.x[which] + b * a.x_sb[which] + s * a.x_ss[which] + h * a.x_sh[which];
    unsigned char* y = a.y[which] + b * a.y_sb[which] + s * a.y_ss[which] + h * a.y_sh[which];
    const float2* cs = table + tt * n;
    constexpr int Z = (int)sizeof(T);
    if (pc >= turned) {
      const int d = 2 * n + (pc - turned) * E;
      if constexpr (VEC) *(u32x4*)(y + d * Z) = *(const u32x4*)(x + d * Z);
      else *(T*)(y + d * Z) = *(const T*)(x + d * Z);
    } else if constexpr (VEC) {
      if (a.interleaved) {
        float v[E];
        Io<T>::unpack(*(const u32x4*)(x + pc * 16), v);
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 f = cs[(pc * E + e) >> 1];
          const float p = v[e], q = v[e + 1];
          v[e] = p * f.x - q * f.y;
          v[e + 1] = q * f.x + p * f.y;
        }
        *(u32x4*)(y + pc * 16) = Io<T>::pack(v);
      } else {
        float p[E], q[E];
        Io<T>::unpack(*(const u32x4*)(x + pc * 16), p);
        Io<T>::unpack(*(const u32x4*)(x + n * Z + pc * 16), q);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float2 f = cs[pc * E + e];
          const float lo = p[e], hi = q[e];
          p[e] = lo * f.x - hi * f.y;
          q[e] = hi * f.x + lo * f.y;
        }
        *(u32x4*)(y + pc * 16) = Io<T>::pack(p);
        *(u32x4*)(y + n * Z + pc * 16) = Io<T>::pack(q);
      }
    } else {
      const int lo = a.interleaved ? 2 * pc : pc, hi = a.interleaved ? 2 * pc + 1 : pc + n;
      const float p = Io<T>::get(x + lo * Z), q = Io<T>::get(x + hi * Z);
      const float2 f = cs[pc];
      Io<T>::put(y + lo * Z, p * f.x - q * f.y);
      Io<T>::put(y + hi * Z, q * f.x + p * f.y);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
using namespace fa::kvhost;

template <typename T>
int launch_rope(const RArgs& a, bool vec, hipStream_t st) {
  const int64_t wgs = ((int64_t)a.tokens + a.per_wg - 1) / a.per_wg;
  const int lds = a.per_wg * a.pairs * 8;
  if (vec) hipLaunchKernelGGL((fa_rope_kernel<T, true>), dim3((unsigned)wgs), dim3(256), lds, st, a);
  else hipLaunchKernelGGL((fa_rope_kernel<T, false>), dim3((unsigned)wgs), dim3(256), lds, st, a);
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int fa_rope_validate(const fa_rope_params* p) { return rope_validate(p); }

int fa_rope_launch(const fa_rope_params* p, void* stream) {
  if (const int rc = rope_validate(p)) return rc;
  if ((int64_t)p->batch * p->seqlen == 0) return FA_OK;
  RArgs a;
  const int64_t z = p->dtype == FA_DTYPE_FP32 ? 4 : 2;
  a.x[0] = (const unsigned char*)p->q; a.x[1] = (const unsigned char*)p->k;
  a.y[0] = (unsigned char*)p->q_out; a.y[1] = (unsigned char*)p->k_out;
  a.positions = p->positions; a.freq = p->inv_freq; a.axes = p->axes;
  a.x_sb[0] = p->q_stride_b * z; a.x_ss[0] = p->q_stride_s * z; a.x_sh[0] = p->q_stride_h * z;
  a.x_sb[1] = p->k_stride_b * z; a.x_ss[1] = p->k_stride_s * z; a.x_sh[1] = p->k_stride_h * z;
  a.y_sb[0] = p->qo_stride_b * z; a.y_ss[0] = p->qo_stride_s * z; a.y_sh[0] = p->qo_stride_h * z;
  a.y_sb[1] = p->ko_stride_b * z; a.y_ss[1] = p->ko_stride_s * z; a.y_sh[1] = p->ko_stride_h * z;
  a.pos_sa = p->pos_stride_a; a.pos_sb = p->pos_stride_b; a.pos_ss = p->pos_stride_s;
  a.tokens = p->batch * p->seqlen; a.seqlen = p->seqlen;
  a.heads[0] = p->heads_q; a.heads[1] = p->heads_k;
  a.head_dim = p->head_dim; a.pairs = p->pairs; a.num_axes = p->num_axes;
  a.positions_64 = p->positions_64; a.freq_64 = p->inv_freq_64; a.interleaved = p->interleaved; a.inverse = p->inverse;
  hipStream_t st = (hipStream_t)stream;
  const bool vec = rope_vector(p);
  a.per_wg = rope_tokens_per_wg(p, vec);
  if (p->dtype == FA_DTYPE_FP32) return launch_rope<float>(a, vec, st);
  return p->dtype == FA_DTYPE_BF16 ? launch_rope<__bf16>(a, vec, st) : launch_rope<_Float16>(a, vec, st);
}

}  // extern "C"
