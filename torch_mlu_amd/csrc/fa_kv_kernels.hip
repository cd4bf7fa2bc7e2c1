// The plan of a serving step and the writes into a paged 8-bit cache: the kernels and the C ABI of fa_kv_plan_* and
// fa_kv_write_* (include/fa_kv.h).
#include <hip/hip_runtime.h>

#include "fa_kv_device.h"
#include "fa_kv_host.h"

namespace {
using namespace fa;

// ---- plan ---------------------------------------------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;

// Inclusive sum over the workgroup's threads of an int64 each; `part` has a place for every wavefront.
__device__ __forceinline__ int64_t wg_scan(int64_t x, int64_t* part, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // the last scan's readers are done
  if (lane == 63) part[wave] = x;
  __syncthreads();
  int64_t before = 0;
  total = 0;
  for (int w = 0; w < (int)blockDim.x / 64; ++w) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  return x + before;
}

// One launch and no meeting of workgroups: each sums all requests' lengths for itself (two scans over at most 8192 numbers,
// which the L2 holds) and then does its share of the tokens, one thread a token, which finds its request by bisection.  The
// token at a page's first position enters the page into the table, so nothing has to go through the requests' pages; entries
// that a thread reads (pages held before) are never those that one writes.
__global__ void __launch_bounds__(kPlanThreads) fa_kv_plan_kernel(const fa_kv_plan_params p) {
  extern __shared__ __attribute__((aligned(16))) int32_t lds[];
  __shared__ int64_t part[kPlanThreads / 64];
  __shared__ int32_t s_taken;
  int32_t* s_end = lds;              // [batch] rows up to and with the request, at most max_tokens
  int32_t* s_page = lds + p.batch;   // [batch] pages given to the requests before; -1: not admitted
  const int tid = threadIdx.x, threads = blockDim.x;
  const int32_t free_count = min(max(*p.free_count, 0), p.free_capacity);
  const int64_t most = (int64_t)p.table_pages * p.page_size;
  if (tid == 0) s_taken = 0;
  int64_t rows_before = 0, pages_before = 0;
  for (int b0 = 0; b0 < p.batch; b0 += threads) {
    const int b = b0 + tid;
    const bool real = b < p.batch;
    const int64_t cached = real ? max(p.cached[b], 0) : 0, add = real ? max(p.new_tokens[b], 0) : 0;
    int64_t rows, pages;
    const int64_t end = rows_before + wg_scan(add, part, rows);
    const bool fits = end <= p.max_tokens && cached + add <= most;
    const uint32_t held = (uint32_t)(min(cached, most) + p.page_size - 1) / (uint32_t)p.page_size;
    const int64_t need = fits ? (int64_t)((uint32_t)(cached + add + p.page_size - 1) / (uint32_t)p.page_size) - held : 0;
    const int64_t taken = pages_before + wg_scan(need, part, pages);
    const bool in = fits && (need == 0 || taken <= free_count);
    if (real) {
      s_end[b] = (int32_t)min(end, (int64_t)p.max_tokens);
      s_page[b] = in ? (int32_t)min(taken - need, (int64_t)0x7fffffff) : -1;
      if (in && need > 0) atomicMax(&s_taken, (int32_t)taken);
      if (blockIdx.x == 0) {
        if (b == 0) p.cu_seqlens[0] = 0;
        p.cu_seqlens[b + 1] = (int32_t)min(end, (int64_t)p.max_tokens);
        p.seqused[b] = (int32_t)min(in ? cached + add : cached, (int64_t)0x7fffffff);
        p.admitted[b] = in ? 1 : 0;
      }
    }
    rows_before += rows;
    pages_before += pages;
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    if (p.batch == 0) p.cu_seqlens[0] = 0;
    *p.free_left = free_count - s_taken;
  }
  const int64_t total = min(rows_before, (int64_t)p.max_tokens);
  for (int64_t t = (int64_t)blockIdx.x * threads + tid; t < p.max_tokens; t += (int64_t)gridDim.x * threads) {
    int32_t pos = 0;
    int64_t slot = -1;
    if (t < total) {
      int lo = 0, hi = p.batch - 1;  // the first request that ends behind t
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_end[mid] > t) hi = mid;
        else lo = mid + 1;
      }
      const int32_t start = lo > 0 ? s_end[lo - 1] : 0, before = s_page[lo];
      const int32_t cached = max(p.cached[lo], 0);
      pos = (int32_t)min((int64_t)cached + (t - start), (int64_t)0x7fffffff);
      if (before >= 0) {
        const uint32_t held = (uint32_t)(cached + (int64_t)p.page_size - 1) / (uint32_t)p.page_size;
        const uint32_t at = (uint32_t)pos / (uint32_t)p.page_size, off = (uint32_t)pos - at * (uint32_t)p.page_size;
        int32_t* row = p.block_table + (int64_t)lo * p.block_table_stride;
        int32_t page;
        if (at < held) {
          page = row[at];
        } else {
          page = p.free_pages[free_count - 1 - before - (int32_t)(at - held)];
          if (off == 0) row[at] = page;
        }
        if (page >= 0) slot = (int64_t)page * p.page_size + off;
      }
    }
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

// ---- writes -------------------------------------------------------------------------------------------------------------
struct WArgs {
  const unsigned char* x[2];  // key, value
  unsigned char* pages[2];
  float* scales[2];
  const int64_t* slots;
  int64_t x_st[2], x_sh[2];               // bytes
  int64_t p_sp[2], p_ss[2], p_sh[2];      // bytes
  int64_t s_sp[2], s_sb[2], s_sh[2];      // elements
  uint32_t n_slots;  // of the pool
  int32_t tokens, heads, head_dim;
  uint32_t scale_block, blocks_per_page;
  int32_t chunk;     // tokens whose runs a wavefront looks for
};

template <typename T>
struct Half;
template <>
struct Half<__bf16> {
  static constexpr unsigned kInf = 0x7f80;
};
template <>
struct Half<_Float16> {
  static constexpr unsigned kInf = 0x7c00;
};

template <int F>
struct Grid8;
template <>
struct Grid8<FA_KV_E4M3> {
  static __device__ __forceinline__ float needed(float amax) {
    // amax = 1.m x 2^k: 448 = 1.75 x 2^8, so e = k - 8, or one more where 1.m > 1.75
    const unsigned u = __builtin_bit_cast(unsigned, amax);
    int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, -100);
    return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
  }
  // four values in the format's range
  static __device__ __forceinline__ unsigned pack(const float* x) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(limit(x[0]), limit(x[1]), 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(limit(x[2]), limit(x[3]), w, true);
  }
  static __device__ __forceinline__ float limit(float x) { return x != x ? x : fminf(fmaxf(x, -448.f), 448.f); }
  static __device__ __forceinline__ void unpack(unsigned w, float* x) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = a[0];
    x[1] = a[1];
    x[2] = b[0];
    x[3] = b[1];
  }
};
template <>
struct Grid8<FA_KV_INT8> {
  static __device__ __forceinline__ float needed(float amax) { return fmaxf(amax * (1.0f / 127), 7.8886091e-31f); }  // 2^-100
  static __device__ __forceinline__ unsigned pack(const float* x) {
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // fmaxf takes its other operand for a NaN; that becomes 0
      const float y = x[i] != x[i] ? 0.f : fminf(fmaxf(rintf(x[i]), -127.f), 127.f);
      w |= ((unsigned)(int)y & 0xffu) << (8 * i);
    }
    return w;
  }
  static __device__ __forceinline__ void unpack(unsigned w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
};

// A wavefront owns (a run of rows that go to one block, a head, key or value): nothing is shared, so the largest magnitude,
// the scale and what has to be rounded again need no atomics, and the result does not depend on an order.  It goes over its
// rows twice, once for the largest magnitude and once to store; the second time they come from the caches.
template <typename T, int F>
__global__ void __launch_bounds__(256) fa_kv_write_kernel(const WArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t per_chunk = 2 * (int64_t)a.heads;
  const int64_t c = unit / per_chunk;
  const int hk = (int)(unit - c * per_chunk), kv = hk >= a.heads ? 1 : 0, h = hk - kv * a.heads;
  const int64_t t_begin = c * a.chunk;
  if (t_begin >= a.tokens) return;

  const int LPR = a.head_dim >> 3, RPI = 64 / LPR;  // lanes of a row (8 elements each), rows an instruction
  const int lr = lane / LPR, lc = lane - lr * LPR;
  const bool mine = lr < RPI;
  const unsigned char* xh = a.x[kv] + (int64_t)h * a.x_sh[kv] + lc * 16;
  unsigned char* ph = a.pages[kv] + (int64_t)h * a.p_sh[kv] + lc * 8;
  float* sh = a.scales[kv] + (int64_t)h * a.s_sh[kv];
  const int64_t x_st = a.x_st[kv], p_ss = a.p_ss[kv], p_sp = a.p_sp[kv];

  auto slot_of = [&](int64_t t) -> uint32_t {  // 0xffffffff: this row goes nowhere
    const int64_t s = a.slots[t];
    return s >= 0 && s < (int64_t)a.n_slots ? (uint32_t)s : 0xffffffffu;
  };
  auto block_of = [&](uint32_t s) -> uint32_t { return s == 0xffffffffu ? s : s / a.scale_block; };

  // runs that begin in this chunk (at most 64 tokens)
  const int64_t t_lane = t_begin + lane;
  const bool inside = lane < a.chunk && t_lane < a.tokens;
  const uint32_t b_lane = inside ? block_of(slot_of(t_lane)) : 0xffffffffu;
  const uint32_t b_before = inside && t_lane > 0 ? block_of(slot_of(t_lane - 1)) : 0xffffffffu;
  uint64_t begins = __ballot(b_lane != 0xffffffffu && b_lane != b_before);
  while (begins) {
    const int first = __builtin_ctzll(begins);
    begins &= begins - 1;
    const int64_t t0 = t_begin + first;
    const uint32_t blk = __builtin_amdgcn_readlane(b_lane, first);
    // how long the run is, and whether it has the block's first row
    int n = 0;
    bool fresh = false;
    for (;;) {
      const int64_t t = t0 + n + lane;
      const uint32_t s = t < a.tokens ? slot_of(t) : 0xffffffffu;
      const bool same = block_of(s) == blk;
      const uint64_t not_same = ~__ballot(same);
      const int k = not_same ? __builtin_ctzll(not_same) : 64;
      fresh = fresh || __ballot(lane < k && s == blk * a.scale_block);
      n += k;
      if (k < 64) break;
    }

    unsigned top = 0;
    for (int i = lr; i < n; i += RPI)
      if (mine) {
        const u32x4 w = *(const u32x4*)(xh + (t0 + i) * x_st);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned lo = w[e] & 0x7fffu, hi = (w[e] >> 16) & 0x7fffu;
          top = max(top, lo < Half<T>::kInf ? lo : 0u);
          top = max(top, hi < Half<T>::kInf ? hi : 0u);
        }
      }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o));
    const float need = Grid8<F>::needed(Mma<T>::to_float((unsigned short)top));

    const uint32_t page = blk / a.blocks_per_page, in_page = blk - page * a.blocks_per_page;
    float* sp = sh + (int64_t)page * a.s_sp[kv] + (int64_t)in_page * a.s_sb[kv];
    const float old = fresh ? 0.f : *sp;
    const float scale = fmaxf(old, need);
    unsigned char* rows = ph + (int64_t)page * p_sp + (int64_t)(in_page * a.scale_block) * p_ss;
    if (!fresh && scale > old) {
      const float f = old / scale;
      for (uint32_t i = lr; i < a.scale_block; i += RPI)
        if (mine) {
          u32x2 w = *(const u32x2*)(rows + (int64_t)i * p_ss);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x[4];
            Grid8<F>::unpack(w[e], x);
#pragma unroll
            for (int z = 0; z < 4; ++z) x[z] *= f;
            w[e] = Grid8<F>::pack(x);
          }
          *(u32x2*)(rows + (int64_t)i * p_ss) = w;
        }
      WAIT_VMCNT(0);  // the rows of this call, which come next, go on top of these stores
    }
    if (lane == 0) *sp = scale;
    const float inv = 1.f / scale;
    for (int i = lr; i < n; i += RPI)
      if (mine) {
        const u32x4 w = *(const u32x4*)(xh + (t0 + i) * x_st);
        const uint32_t at = (uint32_t)a.slots[t0 + i] - blk * a.scale_block;
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[2 * e] = Mma<T>::to_float((unsigned short)(w[e] & 0xffffu)) * inv;
          x[2 * e + 1] = Mma<T>::to_float((unsigned short)(w[e] >> 16)) * inv;
        }
        *(u32x2*)(rows + (int64_t)at * p_ss) = u32x2{Grid8<F>::pack(x), Grid8<F>::pack(x + 4)};
      }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
using namespace fa::kvhost;

template <typename T, int F>
int launch_write(const WArgs& a, hipStream_t st) {
  const int64_t units = ((int64_t)a.tokens + a.chunk - 1) / a.chunk * 2 * a.heads;
  if (units > 0x7fffffffLL * 4) return FA_ERR_UNSUPPORTED;
  hipLaunchKernelGGL((fa_kv_write_kernel<T, F>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int fa_kv_version(void) { return FA_KV_ABI_VERSION; }

const char* fa_kv_error_string(int rc) {
  switch (rc) {
    case FA_OK: return "ok";
    case FA_ERR_BAD_ARG: return "bad argument (null pointer, non-positive size, misaligned pointer or stride, short workspace)";
    case FA_ERR_UNSUPPORTED: return "unsupported shape, size or dtype";
    case FA_ERR_LAUNCH: return "HIP launch failure";
    default: return "unknown error";
  }
}

int fa_kv_plan_validate(const fa_kv_plan_params* p) { return plan_validate(p); }

int fa_kv_plan_launch(const fa_kv_plan_params* p, void* stream) {
  if (const int rc = plan_validate(p)) return rc;
  const int lds = p->batch * 8;
  constexpr auto kfn = fa_kv_plan_kernel;
  if (!ensure_dynamic_lds<kfn>(FA_KV_MAX_BATCH * 8)) return FA_ERR_LAUNCH;
  const int64_t wgs = ((int64_t)p->max_tokens + kPlanThreads - 1) / kPlanThreads;
  hipLaunchKernelGGL(kfn, dim3((unsigned)(wgs < 1 ? 1 : (wgs > 256 ? 256 : wgs))), dim3(kPlanThreads), lds, (hipStream_t)stream, *p);
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}

int fa_kv_write_validate(const fa_kv_write_params* p) { return write_validate(p); }

int fa_kv_write_launch(const fa_kv_write_params* p, void* stream) {
  if (const int rc = write_validate(p)) return rc;
  if (p->tokens == 0) return FA_OK;
  WArgs a;
  a.x[0] = (const unsigned char*)p->key; a.x[1] = (const unsigned char*)p->value;
  a.pages[0] = (unsigned char*)p->key_pages; a.pages[1] = (unsigned char*)p->value_pages;
  a.scales[0] = p->key_scales; a.scales[1] = p->value_scales;
  a.slots = p->slots;
  a.x_st[0] = p->key_stride_t * 2; a.x_sh[0] = p->key_stride_h * 2;
  a.x_st[1] = p->value_stride_t * 2; a.x_sh[1] = p->value_stride_h * 2;
  a.p_sp[0] = p->kp_stride_p; a.p_ss[0] = p->kp_stride_s; a.p_sh[0] = p->kp_stride_h;
  a.p_sp[1] = p->vp_stride_p; a.p_ss[1] = p->vp_stride_s; a.p_sh[1] = p->vp_stride_h;
  a.s_sp[0] = p->ks_stride_p; a.s_sb[0] = p->ks_stride_b; a.s_sh[0] = p->ks_stride_h;
  a.s_sp[1] = p->vs_stride_p; a.s_sb[1] = p->vs_stride_b; a.s_sh[1] = p->vs_stride_h;
  a.n_slots = (uint32_t)p->num_pages * (uint32_t)p->page_size;
  a.tokens = p->tokens; a.heads = p->heads; a.head_dim = p->head_dim;
  a.scale_block = (uint32_t)p->scale_block; a.blocks_per_page = (uint32_t)(p->page_size / p->scale_block);
  a.chunk = p->tokens >= 512 ? 32 : 1;
  hipStream_t st = (hipStream_t)stream;
  if (p->dtype == FA_DTYPE_BF16) return p->format == FA_KV_E4M3 ? launch_write<__bf16, FA_KV_E4M3>(a, st) : launch_write<__bf16, FA_KV_INT8>(a, st);
  return p->format == FA_KV_E4M3 ? launch_write<_Float16, FA_KV_E4M3>(a, st) : launch_write<_Float16, FA_KV_INT8>(a, st);
}

}  // extern "C"
