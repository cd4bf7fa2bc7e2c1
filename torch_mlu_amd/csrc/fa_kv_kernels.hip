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
// that a thread reads (pages held before) are never those that one writes.  Bound by latency, three dependent reads and the
// scans: 64 requests of a token each 3.8 us, 1000 requests with 32768 rows 7.5.
__global__ void __launch_bounds__(kPlanThreads) fa_kv_plan_kernel(const fa_kv_plan_params p) {
  extern __shared__ __attribute__((aligned(16))) int32_t lds[];
  __shared__ int64_t part[kPlanThreads / 64];
  __shared__ int32_t s_taken;
  int32_t* s_end = lds;              // [batch] rows up to and with the request, at most max_tokens
  int32_t* s_page = lds + p.batch;   // [batch] pages given to the requests before; -1: not admitted
  int32_t* s_cached = s_page + p.batch;
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
      s_cached[b] = (int32_t)cached;
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
      const int32_t cached = s_cached[lo];
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

// pairs of 16-bit magnitudes
__device__ __forceinline__ unsigned max_pair(unsigned a, unsigned b) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, b)));
}

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
  // four values in the format's range, or NaN
  static __device__ __forceinline__ unsigned pack(const float* x) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  }
  // infinities to the largest
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
    // 1.5 x 2^23 + x is rounded to whole numbers, to nearest even, and has x's low byte as its own.  (The sum must not be
    // contracted with the product that made x, which is rounded first.)
#pragma clang fp contract(off)
    unsigned u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(unsigned, x[i] + 12582912.0f);
    const unsigned lo = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
    return lo | hi;
  }
  // infinities to the largest, NaN to 0
  static __device__ __forceinline__ float limit(float x) { return x != x ? 0.f : fminf(fmaxf(x, -127.f), 127.f); }
  static __device__ __forceinline__ void unpack(unsigned w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
};

// A wavefront owns (a run of rows that go to one block, a head, key or value): nothing is shared, so the largest magnitude,
// the scale and what has to be rounded again need no atomics, and the result does not depend on an order.  Up to 16 KiB of rows
// (64 at head_dim 128) are loaded at once and stay in registers between the search for the largest magnitude and the
// rounding; where blocks may be longer, a workgroup's four wavefronts (W) share those runs that are, and only runs of more than 64
// KiB are read twice.  Finite values cannot leave the format's range, so only runs with an infinity or a NaN, which their largest
// bit pattern shows, limit them.  12000 rows of 8 heads, head_dim 128, bf16 to e4m3: 19 us, 3.9 TB/s read and written (27 when the
// rows were read twice); 64 rows: 5 us, three dependent reads.
template <typename T, int F, int W>
__global__ void __launch_bounds__(256) fa_kv_write_kernel(const WArgs a) {
#pragma clang fp contract(off)
  constexpr int U = kvhost::kWriteLoads;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t unit = W > 1 ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * 4 + wave;
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

  constexpr uint32_t kNone = 0xffffffffu;
  auto usable = [&](int64_t s) -> uint32_t { return s >= 0 && s < (int64_t)a.n_slots ? (uint32_t)s : kNone; };  // kNone: goes nowhere
  auto block_of = [&](uint32_t s) -> uint32_t { return s == kNone ? s : s / a.scale_block; };

  // Lane l looks at the row l - 1 behind the chunk's first: runs that begin in the chunk (at most 32 rows), and, without a
  // second load, how long they are, if they end within the next 31 rows.
  const int64_t t_lane = t_begin - 1 + lane;
  const uint32_t s_lane = t_lane >= 0 && t_lane < a.tokens ? usable(a.slots[t_lane]) : kNone;
  const uint32_t b_lane = block_of(s_lane);
  const uint32_t b_before = (uint32_t)__shfl_up((int)b_lane, 1);
  uint64_t begins = __ballot(lane >= 1 && lane <= a.chunk && b_lane != kNone && b_lane != b_before);
  int turn = 0;
  while (begins) {
    const int first = __builtin_ctzll(begins);
    begins &= begins - 1;
    const int64_t t0 = t_begin - 1 + first;
    const uint32_t blk = __builtin_amdgcn_readlane(b_lane, first);
    // how long the run is, and whether it has the block's first row
    const uint64_t same = __ballot(b_lane == blk) >> first;
    int n = ~same ? __builtin_ctzll(~same) : 64;  // (zeros come in at the top)
    bool fresh = __ballot(s_lane == blk * a.scale_block && lane >= first && lane < first + n) != 0;
    if (first + n == 64) {  // it may go on
      for (;;) {
        const int64_t t = t0 + n + lane;
        const uint32_t s = t < a.tokens ? usable(a.slots[t]) : kNone;
        const uint64_t other = ~__ballot(block_of(s) == blk);
        const int k = other ? __builtin_ctzll(other) : 64;
        fresh = fresh || __ballot(lane < k && s == blk * a.scale_block);
        n += k;
        if (k < 64) break;
      }
    }
    // Long runs are shared by the workgroup's wavefronts, which all look at the same ones; those that fit one wavefront go round.
    const bool shared = W > 1 && n > U * RPI;
    if (W > 1 && !shared && (turn++ & (W - 1)) != wave) continue;
    const int rw = shared ? W : 1, wr = shared ? wave : 0;  // wavefronts of the run, this one among them
    const uint32_t page = blk / a.blocks_per_page, in_page = blk - page * a.blocks_per_page;
    float* sp = sh + (int64_t)page * a.s_sp[kv] + (int64_t)in_page * a.s_sb[kv];
    float old = !fresh && wr == 0 ? *sp : 0.f;  // (the one that also writes it)

    const int piece = U * RPI * rw;  // rows at once
    u32x4 x[U];
    uint32_t at[U];
    auto load = [&](int base) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u] = u32x4{0, 0, 0, 0};
        at[u] = 0;
        if (base + (u * rw + wr) * RPI >= n) continue;  // (uniform)
        const int row = base + (u * rw + wr) * RPI + lr;
        if (mine && row < n) {
          x[u] = *(const u32x4*)(xh + (t0 + row) * x_st);
          at[u] = (uint32_t)a.slots[t0 + row];
        }
      }
    };
    auto over_run = [&](unsigned x) {  // the largest of all lanes' pairs
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) x = max_pair(x, (unsigned)__shfl_xor((int)x, o));
      x = max(x & 0xffffu, x >> 16);
      if constexpr (W > 1) if (shared) {
        __shared__ unsigned tops[W];
        __shared__ float before;
        __syncthreads();  // the last exchange's readers are done
        if (lane == 0) tops[wave] = x;
        if (threadIdx.x == 0) before = old;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; ++w) x = max(x, tops[w]);
        old = before;
      }
      return x;
    };
    unsigned top = 0;
    for (int base = 0; base < n; base += piece) {
      load(base);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max_pair(top, x[u][e] & 0x7fff7fffu);
    }
    top = over_run(top);
    const bool odd = top >= Half<T>::kInf;
    if (odd) {  // once more, without what is not finite
      top = 0;
      for (int base = 0; base < n; base += piece) {
        if (n > piece) load(base);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned lo = x[u][e] & 0x7fffu, hi = (x[u][e] >> 16) & 0x7fffu;
            top = max_pair(top, (lo < Half<T>::kInf ? lo : 0u) | (hi < Half<T>::kInf ? hi << 16 : 0u));
          }
      }
      top = over_run(top);
    }
    const float need = Grid8<F>::needed(Mma<T>::to_float((unsigned short)top));
    const float scale = fmaxf(old, need);
    unsigned char* rows = ph + (int64_t)page * p_sp + (int64_t)(in_page * a.scale_block) * p_ss;
    if (!fresh && scale > old) {
      const float f = old / scale;
      for (uint32_t i = wr * RPI + lr; i < a.scale_block; i += rw * RPI)
        if (mine) {
          u32x2 w = *(const u32x2*)(rows + (int64_t)i * p_ss);
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float y[4];
            Grid8<F>::unpack(w[e], y);
#pragma unroll
            for (int z = 0; z < 4; ++z) y[z] = Grid8<F>::limit(y[z] * f);
            w[e] = Grid8<F>::pack(y);
          }
          *(u32x2*)(rows + (int64_t)i * p_ss) = w;
        }
      WAIT_VMCNT(0);  // the rows of this call, which come next, go on top of these stores
      if constexpr (W > 1) if (shared) __syncthreads();
    }
    if (lane == 0 && wr == 0) *sp = scale;
    const float inv = 1.f / scale;
    for (int base = 0; base < n; base += piece) {
      if (n > piece) load(base);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (base + (u * rw + wr) * RPI >= n) break;  // (uniform)
        float y[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[2 * e] = Mma<T>::to_float((unsigned short)(x[u][e] & 0xffffu)) * inv;
          y[2 * e + 1] = Mma<T>::to_float((unsigned short)(x[u][e] >> 16)) * inv;
        }
        if (odd) {
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = Grid8<F>::limit(y[e]);
        }
        if (mine && base + (u * rw + wr) * RPI + lr < n)
          *(u32x2*)(rows + (int64_t)(at[u] - blk * a.scale_block) * p_ss) = u32x2{Grid8<F>::pack(y), Grid8<F>::pack(y + 4)};
      }
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
using namespace fa::kvhost;

template <typename T, int F>
int launch_write(const WArgs& a, int64_t wgs, int waves, hipStream_t st) {
  if (waves > 1) hipLaunchKernelGGL((fa_kv_write_kernel<T, F, 4>), dim3((unsigned)wgs), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((fa_kv_write_kernel<T, F, 1>), dim3((unsigned)wgs), dim3(256), 0, st, a);
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
  const int lds = p->batch * 12;
  constexpr auto kfn = fa_kv_plan_kernel;
  if (!ensure_dynamic_lds<kfn>(FA_KV_MAX_BATCH * 12)) return FA_ERR_LAUNCH;
  // few requests leave most of a large workgroup idle in the scans, and its barriers cost
  const int threads = p->batch <= 256 ? 256 : kPlanThreads;
  const int64_t wgs = ((int64_t)p->max_tokens + threads - 1) / threads;
  hipLaunchKernelGGL(kfn, dim3((unsigned)(wgs < 1 ? 1 : (wgs > 256 ? 256 : wgs))), dim3(threads), lds, (hipStream_t)stream, *p);
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
  a.chunk = write_chunk(p);
  const int waves = write_waves(p);
  const int64_t wgs = write_wgs(p);
  hipStream_t st = (hipStream_t)stream;
  if (p->dtype == FA_DTYPE_BF16) return p->format == FA_KV_E4M3 ? launch_write<__bf16, FA_KV_E4M3>(a, wgs, waves, st) : launch_write<__bf16, FA_KV_INT8>(a, wgs, waves, st);
  return p->format == FA_KV_E4M3 ? launch_write<_Float16, FA_KV_E4M3>(a, wgs, waves, st) : launch_write<_Float16, FA_KV_INT8>(a, wgs, waves, st);
}

}  // extern "C"
