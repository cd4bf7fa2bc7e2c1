// Attention over a paged cache of 8-bit values with a scale for each (block of tokens, kv head): the kernels and the C ABI of
// fa_kv_attn_* (include/fa_kv.h).
//
//   S = Q K^T,  score = scale ks S,  P = exp(score - m),  O = sum_j P_j vs_j V_j / sum_j P_j,  lse = m + ln sum_j P_j
//
// K and V enter the matrix cores as bf16 / fp16, which hold every stored value exactly, and the scales of a block are one number
// for 32 keys: ks multiplies the scores' exp2 factor, vs the probabilities before they are rounded.
#include <hip/hip_runtime.h>

#include "fa_fwd_common.h"
#include "fa_kv_device.h"
#include "fa_kv_host.h"

namespace {
using namespace fa;

struct AArgs {
  const unsigned char* q;
  const unsigned char* k;
  const unsigned char* v;
  const float* ks;
  const float* vs;
  unsigned char* out;
  float* lse;
  const int32_t* table;
  const int32_t* used;
  const int32_t* cu_q;
  int64_t q_sb, q_ss, q_sh;  // bytes
  int64_t k_sp, k_ss, k_sh;
  int64_t v_sp, v_ss, v_sh;
  int64_t ks_sp, ks_sb, ks_sh;  // elements
  int64_t vs_sp, vs_sb, vs_sh;
  int64_t o_sb, o_ss, o_sh;        // bytes
  int64_t lse_sb, lse_sh, lse_ss;  // elements
  int64_t bt_stride;
  int32_t batch, heads_q, heads_k, group;
  int32_t seqlen_q, total_q, head_dim;
  int32_t num_pages, table_pages, page_size;
  int32_t page_blocks;      // 32-row blocks of a page
  uint32_t scale_inv;       // ceil(2^31 / n) for scale blocks of n 32-row blocks: (block in the page * scale_inv) >> 31 is its scale
  int32_t is_causal, neg_scale, n_splits;
  int32_t hw_log2;          // streaming kernel: log2 of the heads of a workgroup
  int32_t row_blocks;       // tile kernel: of a sequence; packed calls: places for the blocks of all sequences
  float scale_log2;
  int64_t rows_q;  // query rows of all sequences
  float* ws_o;     // [query rows of all sequences][heads_q][n_splits][head_dim]
  float* ws_ml;    // [...][2]: maximum (log2 domain), sum
};

// Probabilities (at most 1) times this go into the second product: fp16 has 2^-14 as its smallest normal value, and a block
// whose scale is far below the largest, or a key whose probability is, should not fall below it.
template <typename T>
constexpr float kLift = 1.0f;
template <>
constexpr float kLift<_Float16> = 32768.0f;
// ... where a probability may be up to 2^kLazyLog2
template <typename T>
constexpr float kLazyLift = 1.0f;
template <>
constexpr float kLazyLift<_Float16> = 128.0f;

// e4m3's NaN (0x7f and 0xff) among the bytes of w, which become 0; returns whether there were any.  V is searched where a mask
// hides some of its keys: hidden ones have a probability of 0, and 0 x NaN is NaN.  A row that does see such a key is NaN.
__device__ __forceinline__ bool take_nan(unsigned& w) {
  const unsigned t = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // 0x80 for each
  w &= ~((t << 1) - (t >> 7));
  return t != 0;
}

// A wavefront streams 32-key blocks straight into registers, in the layouts that v_mfma_f32_16x16x32 wants:
//   S^T (keys x rows) = K Q^T: lane (L, G) = (lane & 15, lane >> 4) holds DP / 4 bytes of key L from DP / 4 * G on, which are
//     its part of every step of the contraction; Q is laid out to match, as the order of a contraction is free.
//   O^T (d x rows) = V^T P^T: lane (L, G) holds bytes VB L ... VB L + VB - 1 of the 8 keys 4 G + j and 16 + 4 G + j, j < 4,
//     which are the keys of its own scores, so P needs no exchange; byte i of a lane goes to the product that makes rows
//     d = VB L + i, and two keys' bytes are put side by side before they are converted.
// So K and V pass through no LDS, and a wavefront's next block is on its way while it computes.  Bound by reading the cache: 64
// sequences of 8192 keys, 32 / 8 heads, head_dim 128, e4m3: 188 us, 5.5 TB/s.  What was tried for it and changed nothing: two
// blocks on their way a wavefront (twice the registers, half the wavefronts), K pieces in whole cache lines an instruction.
//
// A row of a token and head has only 128 bytes at head_dim 128, and memory is read at its full rate only where neighbours
// are read together (64 sequences of 8192 keys, 8 kv heads: 204 us a head a workgroup, 182 with one kv head in the cache): half
// of a workgroup's wavefronts take the neighbouring head of the same blocks.  Those of one head take turns in the blocks, and
// meet in LDS at the end.
template <typename T, int F, int DP, int CT, int NW>
__global__ void __launch_bounds__(NW * 64, CT == 1 && DP <= 128 ? 4 : (DP <= 128 ? 2 : 1)) fa_kv_attn_kernel(const AArgs a) {
  constexpr int KC = DP / 64;  // 16-byte pieces of a key a lane holds
  constexpr int KS = DP / 32;  // steps of the contraction over head_dim
  constexpr int VB = DP / 16;  // bytes of a key of V a lane holds = 16-row blocks of O^T
  constexpr int VW = VB / 4;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int L = lane & 15, G = lane >> 4;
  const int hw = 1 << a.hw_log2, turns = NW >> a.hw_log2, turn = wave >> a.hw_log2;

  const unsigned groups = (unsigned)a.heads_k >> a.hw_log2;
  const unsigned unit = blockIdx.x / (unsigned)a.n_splits;
  const int split = (int)(blockIdx.x - unit * (unsigned)a.n_splits);
  const int b = (int)(unit / groups), hk0 = (int)(unit - (unsigned)b * groups) << a.hw_log2;
  const int hk = hk0 + (wave & (hw - 1));

  // the first table entry, asked for before it is known whether the sequence has that key
  ConstI32Ptr tbl = (ConstI32Ptr)(uintptr_t)(a.table + (int64_t)b * a.bt_stride);
  const int blk0 = split * turns + turn, stride = a.n_splits * turns;
  const int first_idx = blk0 / a.page_blocks, first_in = blk0 - first_idx * a.page_blocks;
  const int first_page = first_idx < a.table_pages ? tbl[first_idx] : 0;
  const QRows rows = query_rows(a.cu_q, b, a.seqlen_q, a.total_q);
  const int R = rows.count * a.group;  // at most 16 CT
  if (R <= 0) return;
  const int Lk = min(max(a.used[b], 0), a.table_pages * a.page_size);
  const int last_q = (R - 1) / a.group;
  // row i of the sequence sees keys up to shift + i
  const int shift = a.is_causal ? Lk - rows.aligned : 0x3fffffff;
  const int mask_from = min(Lk, shift + 1);  // first key that some row does not see
  const int keys = min(Lk, max(shift + last_q + 1, 0));

  // Every n-th 32-key block is this wavefront's: slices of a sequence are equally long whatever its length, and which table
  // entry comes first does not wait for it.
  const int nblk = (keys + 31) >> 5;
  const int n_my = max(0, (nblk - blk0 + stride - 1) / stride);

  int lim[CT];  // the last key that this lane's row sees
  s16x8 qf[CT][KS];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int r = 16 * ct + L;
    const int qr = min(r, R - 1) / a.group, g = min(r, R - 1) - qr * a.group;
    lim[ct] = min(Lk - 1, shift + qr);
    const unsigned char* qp = a.q + (a.cu_q ? 0 : (int64_t)b * a.q_sb) + (int64_t)(rows.first + qr) * a.q_ss + (int64_t)(hk * a.group + g) * a.q_sh;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = 16 * KC * G + 8 * s;
      u32x4 x = {0, 0, 0, 0};
      if (r < R && d < a.head_dim) x = *(const u32x4*)(qp + d * 2);
      if (a.neg_scale) x ^= 0x80008000u;
      qf[ct][s] = __builtin_bit_cast(s16x8, x);
    }
  }

  f32x4 o[VB][CT];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int i = 0; i < VB; ++i) o[i][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // O is held in units of `ref`, the largest V scale so far, so that P vs / ref stays in fp16's range whatever the scales are
  float ref = 1.17549435e-38f;
  int poison = 0;  // bit ct: this lane's row sees a NaN of V among its keys

  if (n_my > 0) {
    const unsigned char* kh = a.k + (int64_t)hk * a.k_sh;
    const unsigned char* vh = a.v + (int64_t)hk * a.v_sh;
    ConstF32Ptr ksp = (ConstF32Ptr)(uintptr_t)(a.ks + (int64_t)hk * a.ks_sh);
    ConstF32Ptr vsp = (ConstF32Ptr)(uintptr_t)(a.vs + (int64_t)hk * a.vs_sh);
    const unsigned kss = (unsigned)a.k_ss, vss = (unsigned)a.v_ss;
    const int stride_idx = stride / a.page_blocks, stride_in = stride - stride_idx * a.page_blocks;
    int kd[KC];
#pragma unroll
    for (int c = 0; c < KC; ++c) kd[c] = 16 * (KC * G + c) < a.head_dim ? 16 * (KC * G + c) : 0;
    const int vd = VB * L < a.head_dim ? VB * L : 0;

    int pg_idx = first_idx, pg_in = first_in, page = first_page;

    struct Block {
      const unsigned char* k;
      const unsigned char* v;
      int left;      // last row that exists
      bool hidden;   // its table entry names no page
      float ks, vs;
    };
    // this wavefront's next block; the table entry of the one after it is requested
    auto next_block = [&](int blk, bool more) __attribute__((always_inline)) -> Block {
      Block x;
      x.hidden = (unsigned)page >= (unsigned)a.num_pages;
      const int64_t p = x.hidden ? 0 : page;
      const unsigned row = (unsigned)pg_in * 32u;
      const int64_t sb = (int64_t)(((uint64_t)(unsigned)pg_in * a.scale_inv) >> 31);
      x.k = kh + p * a.k_sp + (uint64_t)row * kss;
      x.v = vh + p * a.v_sp + (uint64_t)row * vss;
      x.ks = ksp[p * a.ks_sp + sb * a.ks_sb];
      x.vs = x.hidden ? 0.f : vsp[p * a.vs_sp + sb * a.vs_sb];
      x.left = Lk - 1 - blk * 32;
      pg_in += stride_in;
      pg_idx += stride_idx;
      if (pg_in >= a.page_blocks) {
        pg_in -= a.page_blocks;
        ++pg_idx;
      }
      if (more) page = tbl[pg_idx];
      return x;
    };

    u32x4 kr[2][KC];
    unsigned vr[8][VW];
    // Rows behind the sequence's last one are that one again.  Addresses are clamped in every block rather than in a branch for
    // the last: with loads in branches the compiler cannot tell how many are on their way, and waits for too many.
    auto load_k = [&](const Block& x) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const unsigned row = __umul24((unsigned)min(16 * t + L, x.left), kss);
#pragma unroll
        for (int c = 0; c < KC; ++c) kr[t][c] = *(const u32x4*)(x.k + (row + kd[c]));
      }
      __builtin_amdgcn_sched_barrier(0);  // loads stay in their order, for the same reason
    };
    auto load_v = [&](const Block& x) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const unsigned char* p = x.v + (__umul24((unsigned)min(4 * G + (j < 4 ? j : 12 + j), x.left), vss) + vd);
        if constexpr (VW == 1) {
          vr[j][0] = *(const unsigned*)p;
        } else if constexpr (VW == 2) {
          const u32x2 y = *(const u32x2*)p;
          vr[j][0] = y[0];
          vr[j][1] = y[1];
        } else {
          const u32x4 y = *(const u32x4*)p;
#pragma unroll
          for (int i = 0; i < 4; ++i) vr[j][i] = y[i];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };

    auto step = [&](const Block& x, int blk, auto&& after_k, auto&& after_v) __attribute__((always_inline)) {
      f32x4 s[2][CT];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) s[t][ct] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const unsigned w0 = kr[t][ks >> 1][2 * (ks & 1)], w1 = kr[t][ks >> 1][2 * (ks & 1) + 1];
          const u32x4 f = {Stored<T, F>::template pair<0>(w0), Stored<T, F>::template pair<1>(w0),
                           Stored<T, F>::template pair<0>(w1), Stored<T, F>::template pair<1>(w1)};
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) s[t][ct] = Mma<T>::m16(__builtin_bit_cast(s16x8, f), qf[ct][ks], s[t][ct]);
        }
      after_k();

      // scale 0 (and a K scale of 0) must not meet the -inf of a masked score
      const float c = fmaxf(a.scale_log2 * x.ks, 1e-30f);
      if (blk * 32 + 32 > mask_from || x.hidden) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int lm = x.hidden ? -1 : lim[ct] - blk * 32 - 4 * G;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if (e > lm) s[0][ct][e] = -INFINITY;
            if (16 + e > lm) s[1][ct][e] = -INFINITY;
          }
        }
        if constexpr (F == FA_KV_E4M3) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < VW; ++i) any |= take_nan(vr[j][i]);
            const bool bad = ((__ballot(any) >> (16 * G)) & 0xffffu) != 0;  // the 16 lanes of a G hold the same keys
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              if (bad && !x.hidden && (j < 4 ? j : 12 + j) <= lim[ct] - blk * 32 - 4 * G) poison |= 1 << ct;
          }
        }
      }
      if (x.vs > ref) {  // wavefront-uniform and rare
        const float f = ref / x.vs;
        ref = x.vs;
#pragma unroll
        for (int i = 0; i < VB; ++i)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) o[i][ct] *= f;
      }
      const float vf = x.vs / ref * kLift<T>;
      if (x.hidden) {  // what was loaded in its place must not meet a probability of 0: it may be NaN
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int i = 0; i < VW; ++i) vr[j][i] = 0;
      }
      s16x8 pb[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        // (the compiler waits for the matrix pipe only in front of instructions it knows: each product is first read by a
        // canonicalize, and the asm maxima depend on it)
        const float g0 = __builtin_canonicalizef(s[0][ct][3]), g1 = __builtin_canonicalizef(s[1][ct][3]);
        float mx = max3d(s[0][ct][0], s[0][ct][1], s[0][ct][2], g0);
        mx = max3(mx, g0, max3d(s[1][ct][0], s[1][ct][1], s[1][ct][2], g1));
        mx = max2(mx, g1) * c;
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = pair_max32(mx);
        if (__any(mx > m[ct])) {
          const float mn = fmaxf(m[ct], mx);
          const float f = mn == -INFINITY ? 1.f : fast_exp2(m[ct] - mn);
          m[ct] = mn;
          l[ct] *= f;
#pragma unroll
          for (int i = 0; i < VB; ++i) o[i][ct] *= f;
        }
        const float base = m[ct] == -INFINITY ? 0.f : m[ct];
        float p[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = fast_exp2(s[0][ct][e] * c - base);
          p[4 + e] = fast_exp2(s[1][ct][e] * c - base);
          l[ct] += p[e] + p[4 + e];
        }
        u32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = Mma<T>::pack2(p[2 * e] * vf, p[2 * e + 1] * vf);
        pb[ct] = __builtin_bit_cast(s16x8, y);
      }

#pragma unroll
      for (int wd = 0; wd < VW; ++wd)
        static_for<0, 2>([&](auto H) {
          constexpr int h = decltype(H)::value;
          u32x4 fa, fb;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            // (key 2t, key 2t + 1) of byte 2h, then of byte 2h + 1
            const unsigned z = __builtin_amdgcn_perm(vr[2 * t + 1][wd], vr[2 * t][wd], h ? 0x07030602u : 0x05010400u);
            fa[t] = Stored<T, F>::template pair<0>(z);
            fb[t] = Stored<T, F>::template pair<1>(z);
          }
          constexpr int i0 = 2 * h;
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            o[4 * wd + i0][ct] = Mma<T>::m16(__builtin_bit_cast(s16x8, fa), pb[ct], o[4 * wd + i0][ct]);
            o[4 * wd + i0 + 1][ct] = Mma<T>::m16(__builtin_bit_cast(s16x8, fb), pb[ct], o[4 * wd + i0 + 1][ct]);
          }
        });
      after_v();
    };

    Block x = next_block(blk0, n_my > 1);
    load_k(x);
    load_v(x);
    int blk = blk0;
    for (int it = 0; it + 1 < n_my; ++it, blk += stride) {
      const Block y = next_block(blk + stride, it + 2 < n_my);
      step(x, blk, [&] { load_k(y); }, [&] { load_v(y); });
      x = y;
    }
    step(x, blk, [] {}, [] {});
  }

  // ---- the wavefronts' partials, 16 rows at a time ----
  constexpr int OS = DP + 4;
  float* so = (float*)smem;                        // [NW][16][OS]
  float* sml = (float*)(smem + NW * 16 * OS * 4);  // [NW][16][2]
  poison |= __shfl_xor(poison, 16);
  poison |= __shfl_xor(poison, 32);
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (16 * ct >= R) break;
    const float o_unit = (poison >> ct) & 1 ? __builtin_nanf("") : ref / kLift<T>;
    float ls = l[ct];
    ls += __shfl_xor(ls, 16);
    ls = pair_sum32(ls);
    if (ct) __syncthreads();
    float* row = so + (wave * 16 + L) * OS;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int i = 0; i < VB; i += 4) {
        f32x4 y;
#pragma unroll
        for (int z = 0; z < 4; ++z) y[z] = o[i + z][ct][e] * o_unit;
        *(f32x4*)(row + VB * (4 * G + e) + i) = y;
      }
    if (G == 0) {
      sml[(wave * 16 + L) * 2] = m[ct];
      sml[(wave * 16 + L) * 2 + 1] = ls;
    }
    __syncthreads();
    const int nrows = min(16, R - 16 * ct);
    constexpr int TPR = DP / 4;
    for (int item = tid; item < hw * nrows * TPR; item += NW * 64) {
      const int hi = item / TPR, d = (item % TPR) * 4;
      const int hh = hi / nrows, i = hi - hh * nrows;
      float M = -INFINITY;
      for (int y = 0; y < turns; ++y) M = fmaxf(M, sml[((y * hw + hh) * 16 + i) * 2]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.f;
      for (int y = 0; y < turns; ++y) {
        const int at = (y * hw + hh) * 16 + i;
        const float ly = sml[at * 2 + 1];
        if (ly == 0.f) continue;  // a wavefront that saw no key of this row (a NaN goes on to the result)
        const float f = fast_exp2(sml[at * 2] - M);
        sum += ly * f;
        acc += *(const f32x4*)(so + at * OS + d) * f;
      }
      const int r = 16 * ct + i, qr = r / a.group, h = (hk0 + hh) * a.group + r - qr * a.group;
      if (a.n_splits == 1) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        if (d < a.head_dim) {
          unsigned char* p = a.out + (a.cu_q ? 0 : (int64_t)b * a.o_sb) + (int64_t)(rows.first + qr) * a.o_ss + (int64_t)h * a.o_sh + d * 2;
          *(u32x2*)p = u32x2{Mma<T>::pack2(acc[0] * inv, acc[1] * inv), Mma<T>::pack2(acc[2] * inv, acc[3] * inv)};
        }
        if (d == 0)
          a.lse[(a.cu_q ? 0 : (int64_t)b * a.lse_sb) + (int64_t)h * a.lse_sh + (int64_t)(rows.first + qr) * a.lse_ss] =
              sum != 0.f ? (M + __builtin_log2f(sum)) * kLn2 : INFINITY;
      } else {
        const int64_t slot = ((rows.place + qr) * a.heads_q + h) * a.n_splits + split;
        if (d < a.head_dim) *(f32x4*)(a.ws_o + slot * a.head_dim + d) = acc;
        if (d == 0) *(f32x2*)(a.ws_ml + slot * 2) = f32x2{M, sum};
      }
    }
  }
}

// A copy of a kernel argument that the compiler takes for a value of its own: loaded in groups of eight, arguments are also kept
// (and spilled) in groups of eight.
__device__ __forceinline__ unsigned own(unsigned x) {
  asm volatile("" : "+s"(x));
  return x;
}
// The arguments once more, read where they are used: what the end needs is not kept through the loop.
typedef const __attribute__((address_space(4))) AArgs* ArgsPtr;
__device__ __forceinline__ ArgsPtr args_again() {
  ArgsPtr p = (ArgsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// Many rows against the cache, more than 32 a kv head (chunks of prompts, packed batches): MFMA-bound.  One workgroup owns 128
// (query row, head of the group) pairs of one (sequence, kv head), 32 a wavefront, and goes through the keys in tiles of 64.  A
// tile is loaded into registers while the one before it is computed, converted once for all four wavefronts and kept in LDS as bf16 / fp16, double
// buffered; S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_32x32x16 with one lane a row, as in the 16-bit tile kernel, whose LDS
// layouts these are.  The heads of a group share the tile, so a conversion serves 4 x 32 rows instead of one wavefront's.
// Bound by the issue of matrix and vector instructions, which add up: 500 rows over 32768 keys, 32 / 8 heads, head_dim 128, e4m3:
// 321 us with the join of 4 slices, 831 TFLOP/s; a wavefront's tile is 32 products (1000 cycles) and about 240 vector
// instructions (1200), of which the conversion, 32 + 8 stores, is a sixth; both together take 2400.
template <typename T, int F, int DP>
__global__ void __launch_bounds__(256, DP <= 128 ? 2 : 1) fa_kv_tile_kernel(const AArgs a) {
  constexpr int ROWB = DP * 2;        // bytes of a row in LDS
  constexpr int BM = 128, BN = 64;
  constexpr int TILE = BN * ROWB;
  constexpr int KS = DP / 16;         // steps of the contraction over head_dim
  constexpr int MB = DP / 32;         // 32-row blocks of O^T
  constexpr int PPR = DP / 16;        // 16-byte pieces of a stored row
  constexpr int RPP = 256 / PPR;      // rows a pass of the workgroup loads
  constexpr int NP = BN / RPP;        // passes a tile
  constexpr int CPR = DP / 8;         // 16-byte chunks of a row in LDS
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];  // K0 K1 V0 V1

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5, c32 = lane & 31;

  int b, hk, split, rb;
  if (a.cu_q) {
    // The sequences' blocks of 128 rows share the grid without a place for blocks that a shorter one has not (a workgroup that
    // exits takes its LDS for a microsecond or two, and the ones behind it wait).  Up to 64 sequences: the blocks one after the
    // other, those of few rows (single tokens) behind all others, where they fill the gaps of the last round (16 x 512 over
    // 4096 213 -> 178 us in one slice, 16 / 16 heads, 6 x 2000 over 4000 143 -> 130).  More: with c rows before it, sequence b begins at
    // place c * group / 128 + b, which leaves room for its blocks and at most one place too many.
    const unsigned nhs = (unsigned)(a.heads_k * a.n_splits);
    unsigned hs, place;
    if (nhs % 8 == 0) {  // a head's blocks on one XCD, one place of all its heads and slices after the other (head by head the
                         // last slice's long blocks began when the rest was done: 16 x 512 over 4096, 194 us instead of 181)
      place = (blockIdx.x >> 3) / (nhs >> 3);
      hs = ((blockIdx.x >> 3) - place * (nhs >> 3)) * 8 + (blockIdx.x & 7);
    } else {
      place = blockIdx.x / nhs;
      hs = blockIdx.x - place * nhs;
    }
    if (a.batch <= 64) {  // lane i looks at sequence i
      const QRows of_lane = query_rows(a.cu_q, min(lane, a.batch - 1), a.seqlen_q, a.total_q);
      const unsigned R = lane < a.batch ? (unsigned)of_lane.count * (unsigned)a.group : 0, n = (R + BM - 1) / BM;
      const bool few = R > 0 && R <= 32;  // one wavefront's
      unsigned end = few ? 0 : n;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const unsigned y = (unsigned)__shfl_up((int)end, d);
        if (lane >= d) end += y;
      }
      const uint64_t fews = __ballot(few);
      const unsigned others = (unsigned)__builtin_amdgcn_readlane((int)end, 63);
      const unsigned first = few ? others + (unsigned)__popcll(fews & ((1ULL << lane) - 1)) : end - n;
      const uint64_t here = __ballot(place >= first && place - first < n);
      if (!here) return;
      b = __builtin_ctzll(here);
      rb = (int)(place - (unsigned)__builtin_amdgcn_readlane((int)first, b));
    } else {
      ConstI32Ptr cu = (ConstI32Ptr)(uintptr_t)a.cu_q;
      auto begin = [&](int i) { return (unsigned)((uint64_t)min(max(cu[i], 0), a.total_q) * (unsigned)a.group / BM) + (unsigned)i; };
      int lo = 0, hi = a.batch - 1;  // the last sequence that begins at or before this place
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (begin(mid) <= place) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      rb = (int)(place - begin(lo));
    }
    hk = (int)(hs / (unsigned)a.n_splits);
    split = (int)(hs - (unsigned)hk * a.n_splits);
  } else {
    // consecutive workgroups go round the 8 XCDs: those that share K and V (the row blocks of one sequence, head and slice) are
    // neighbours on one, and a sequence's heads, whose lengths are the same, are spread over all
    const unsigned turn = (blockIdx.x >> 3) / (unsigned)a.row_blocks;
    const unsigned unit = turn * 8 + (blockIdx.x & 7);
    const unsigned bhk = unit / (unsigned)a.n_splits;
    rb = (int)((blockIdx.x >> 3) - turn * a.row_blocks);
    split = (int)(unit - bhk * a.n_splits);
    b = (int)(bhk / (unsigned)a.heads_k);
    hk = (int)(bhk - (unsigned)b * a.heads_k);
    if (b >= a.batch) return;
  }

  const QRows rows = query_rows(a.cu_q, b, a.seqlen_q, a.total_q);
  const int R = rows.count * a.group, blocks = (R + BM - 1) / BM;
  if ((unsigned)rb >= (unsigned)blocks) return;
  const int m0 = (blocks - 1 - rb) * BM;  // the one with the most keys first
  const int Lk = min(max(a.used[b], 0), a.table_pages * a.page_size);
  const int shift = a.is_causal ? Lk - rows.aligned : 0x3fffffff;
  const int last_q = (min(m0 + BM, R) - 1) / a.group;
  const int keys = min(Lk, max(shift + last_q + 1, 0));
  const int all_tiles = (keys + BN - 1) / BN;
  const int per_split = (all_tiles + a.n_splits - 1) / a.n_splits;
  const int jt0 = split * per_split, ntiles = min(all_tiles, jt0 + per_split);

  // this lane's row, and the span of its wavefront's
  const int r = m0 + 32 * wave + c32;
  const int qr = min(r, R - 1) / a.group, hg = min(r, R - 1) - qr * a.group;
  const bool wave_live = m0 + 32 * wave < R;
  const int lim_row = min(Lk - 1, shift + qr);
  const int wave_lo = min(Lk - 1, shift + (m0 + 32 * wave) / a.group);                          // last key its first row sees
  const int wave_hi = min(Lk - 1, shift + min(m0 + 32 * wave + 31, R - 1) / a.group);

  // ---- the next tile: pages and scales of its two 32-key halves ----
  // Table entries (of the tile after the next) and scales (of the next) come by vector loads together with K and V, and are
  // moved to scalar registers when those have landed: as scalar loads they share a counter with LDS reads, and every tile
  // began with waiting for them.
  const int32_t* tbl = a.table + (int64_t)b * a.bt_stride;
  const unsigned char* kh = a.k + (int64_t)hk * a.k_sh;
  const unsigned char* vh = a.v + (int64_t)hk * a.v_sh;
  const float* ksp = a.ks + (int64_t)hk * a.ks_sh;
  const float* vsp = a.vs + (int64_t)hk * a.vs_sh;
  const unsigned kss = own((unsigned)a.k_ss), vss = own((unsigned)a.v_ss);
  const unsigned k_sp = own((unsigned)a.k_sp), v_sp = own((unsigned)a.v_sp), ks_sp = own((unsigned)a.ks_sp), vs_sp = own((unsigned)a.vs_sp);
  const unsigned ks_sb = own((unsigned)a.ks_sb), vs_sb = own((unsigned)a.vs_sb), scale_inv = own(a.scale_inv);
  const unsigned num_pages = own((unsigned)a.num_pages);
  const int page_blocks = (int)own((unsigned)a.page_blocks);
  unsigned zero;  // keeps the loads at wavefront-uniform addresses vector loads
  asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
  auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };  // a quotient comes from the vector unit
  const int last_block = max(Lk - 1, 0) >> 5, last_entry = scalar(last_block / page_blocks);
  int nb = 2 * jt0;                                    // the next tile's first 32-key block,
  int nb_idx = scalar(nb / page_blocks), nb_in = nb - nb_idx * page_blocks;  // its entry of the table and place in the page
  int page0 = 0, page1 = 0;                            // the next tile's entries
  bool hid0 = false, hid1 = false;                     // the current tile's: the entry names no page
  bool next_hid0 = false, next_hid1 = false;
  float sk0 = 0.f, sk1 = 0.f, sv0 = 0.f, sv1 = 0.f;    // the current tile's scales
  float nk0 = 0.f, nk1 = 0.f, nv0 = 0.f, nv1 = 0.f;    // the next tile's, in flight
  int in_flight0 = 0, in_flight1 = 0;                  // entries of the tile after that, in flight
  // loads nb's tile and the entries of the one after it
  // (The lambdas that touch register arrays are inlined by force: where one stays a call, as store_tile did for int8 at 256, the
  // arrays live in memory: 16/1 heads of 256, 2x4 rows over 3386 keys 87 us instead of 25.)
  const int pc = tid % PPR, prow = tid / PPR;
  const int pd = pc * 16 < a.head_dim ? pc * 16 : 0;
  u32x4 kraw[NP], vraw[NP];
  auto step_block = [&](int& idx, int& in) {
    if (++in >= page_blocks) {
      in = 0;
      ++idx;
    }
  };
  auto load_entries = [&]() __attribute__((always_inline)) {
    int i1 = nb_idx, in = nb_in;
    step_block(i1, in);
    in_flight0 = *(const int32_t*)((const unsigned char*)(tbl + min(nb_idx, last_entry)) + zero);
    in_flight1 = *(const int32_t*)((const unsigned char*)(tbl + min(i1, last_entry)) + zero);
  };
  auto load_tile = [&]() __attribute__((always_inline)) {
    int idx1 = nb_idx, in1 = nb_in;
    step_block(idx1, in1);
    int left0 = Lk - 1 - nb * 32, left1 = left0 - 32;
    unsigned p0 = (unsigned)page0, p1 = (unsigned)page1;
    unsigned r0 = (unsigned)nb_in, r1 = (unsigned)in1;
    nb += 2;
    nb_idx = idx1;
    nb_in = in1;
    step_block(nb_idx, nb_in);
    load_entries();
    if (left1 < 0) {  // no key in the second half: copies of rows that exist
      left1 = left0;
      p1 = p0;
      r1 = r0;
    }
    next_hid0 = p0 >= num_pages;
    next_hid1 = p1 >= num_pages;
    p0 = next_hid0 ? 0u : p0;
    p1 = next_hid1 ? 0u : p1;
    const unsigned char* k0 = kh + (uint64_t)p0 * k_sp + (uint64_t)(r0 * 32u) * kss;
    const unsigned char* k1 = kh + (uint64_t)p1 * k_sp + (uint64_t)(r1 * 32u) * kss;
    const unsigned char* v0 = vh + (uint64_t)p0 * v_sp + (uint64_t)(r0 * 32u) * vss;
    const unsigned char* v1 = vh + (uint64_t)p1 * v_sp + (uint64_t)(r1 * 32u) * vss;
    // rows behind the sequence's last one are that one again
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const bool second = RPP == 64 ? wave >= 2 : RPP * i >= 32;
      const unsigned row = (unsigned)min((prow + RPP * i) & 31, second ? left1 : left0);
      kraw[i] = *(const u32x4*)((second ? k1 : k0) + (__umul24(row, kss) + pd));
      vraw[i] = *(const u32x4*)((second ? v1 : v0) + (__umul24(row, vss) + pd));
    }
    const unsigned b0 = (unsigned)(((uint64_t)r0 * scale_inv) >> 31), b1 = (unsigned)(((uint64_t)r1 * scale_inv) >> 31);
    nk0 = *(const float*)((const unsigned char*)(ksp + ((uint64_t)p0 * ks_sp + (uint64_t)b0 * ks_sb)) + zero);
    nk1 = *(const float*)((const unsigned char*)(ksp + ((uint64_t)p1 * ks_sp + (uint64_t)b1 * ks_sb)) + zero);
    nv0 = *(const float*)((const unsigned char*)(vsp + ((uint64_t)p0 * vs_sp + (uint64_t)b0 * vs_sb)) + zero);
    nv1 = *(const float*)((const unsigned char*)(vsp + ((uint64_t)p1 * vs_sp + (uint64_t)b1 * vs_sb)) + zero);
  };
  auto uniform = [](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x))); };
  auto arrived = [&]() __attribute__((always_inline)) {  // what was in flight becomes the current tile's, and the next one's entries
    page0 = __builtin_amdgcn_readfirstlane(in_flight0);
    page1 = __builtin_amdgcn_readfirstlane(in_flight1);
    hid0 = next_hid0;
    hid1 = next_hid1;
    sk0 = uniform(nk0);
    sk1 = uniform(nk1);
    sv0 = hid0 ? 0.f : uniform(nv0);
    sv1 = hid1 ? 0.f : uniform(nv1);
  };
  int st_k[NP], st_v[NP];  // LDS offsets of this thread's pieces (the second chunk is at ^ 16)
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int row = prow + RPP * i;
    st_k[i] = row * ROWB + ((2 * pc) ^ swzK<DP>(row)) * 16;
    st_v[i] = 2 * TILE + row * ROWB + ((2 * pc) ^ swzV<DP>(row)) * 16;
  }
  auto convert = [](unsigned w0, unsigned w1) {
    return u32x4{Stored<T, F>::template pair<0>(w0), Stored<T, F>::template pair<1>(w0), Stored<T, F>::template pair<0>(w1),
                 Stored<T, F>::template pair<1>(w1)};
  };
  __shared__ int nan_key[2][BN], nan_tile[2];  // the last tile in which this key (a key) of a buffer had a NaN in V
  if (tid < 2 * BN) (&nan_key[0][0])[tid] = -1;
  if (tid < 2) nan_tile[tid] = -1;
  const int shown = min(Lk - 1, shift + m0 / a.group);  // the last key that all rows of the workgroup see
  auto store_tile = [&](int buf, int j) __attribute__((always_inline)) {
    if (next_hid0 || next_hid1) {  // what was loaded in their place may be NaN, and must not meet a probability of 0
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const bool second = RPP == 64 ? wave >= 2 : RPP * i >= 32;
        if (second ? next_hid1 : next_hid0) vraw[i] = u32x4{0, 0, 0, 0};
      }
    }
    if constexpr (F == FA_KV_E4M3) {
      if (j * BN + BN - 1 > shown) {
#pragma unroll
        for (int i = 0; i < NP; ++i) {
          bool any = false;
#pragma unroll
          for (int z = 0; z < 4; ++z) {
            unsigned y = vraw[i][z];
            any |= take_nan(y);
            vraw[i][z] = y;
          }
          if (any) nan_key[buf][prow + RPP * i] = nan_tile[buf] = j;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      unsigned char* base = smem + buf * TILE;
      *(u32x4*)(base + st_k[i]) = convert(kraw[i][0], kraw[i][1]);
      *(u32x4*)(base + (st_k[i] ^ 16)) = convert(kraw[i][2], kraw[i][3]);
      *(u32x4*)(base + st_v[i]) = convert(vraw[i][0], vraw[i][1]);
      *(u32x4*)(base + (st_v[i] ^ 16)) = convert(vraw[i][2], vraw[i][3]);
    }
  };

  if (ntiles > jt0) {
    load_entries();
    page0 = __builtin_amdgcn_readfirstlane(in_flight0);
    page1 = __builtin_amdgcn_readfirstlane(in_flight1);
    load_tile();
  }

  // ---- Q through the K and V buffers: 64 rows in each pair of them, whole rows an instruction ----
  int kaddr[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) kaddr[ks] = c32 * ROWB + (((2 * ks + g) ^ swzK<DP>(c32)) * 16);
  s16x8 qf[KS];
  {
    const unsigned char* qb = a.q + (a.cu_q ? 0 : (int64_t)b * a.q_sb) + (int64_t)rows.first * a.q_ss + (int64_t)hk * a.group * a.q_sh;
#pragma unroll
    for (int i = 0; i < BM * CPR / 256; ++i) {
      const int row = (i * 256 + tid) / CPR, ch = (i * 256 + tid) % CPR;
      const int rr = min(m0 + row, R - 1), rq = rr / a.group, rh = rr - rq * a.group;
      u32x4 x = {0, 0, 0, 0};
      if (ch * 8 < a.head_dim) x = *(const u32x4*)(qb + (int64_t)rq * a.q_ss + (int64_t)rh * a.q_sh + ch * 16);
      *(u32x4*)(smem + row * ROWB + ((ch ^ swzK<DP>(row)) * 16)) = x;
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      u32x4 x = *(const u32x4*)(smem + 32 * wave * ROWB + kaddr[ks]);
      if (a.neg_scale) x ^= 0x80008000u;
      qf[ks] = __builtin_bit_cast(s16x8, x);
    }
    __syncthreads();
  }

  const int L = lane & 15, G = lane >> 4;
  const int v_row = 4 * g + (L >> 2);
  int vaddr[MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
    vaddr[mb] = v_row * ROWB + (L & 1) * 8 + (((4 * mb + 2 * (G & 1) + ((L & 3) >> 1)) ^ swzV<DP>(v_row)) * 16);
  LDS_AS const unsigned char* kptr[KS];
  LDS_AS const unsigned char* vptr[MB];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    kptr[ks] = (LDS_AS const unsigned char*)smem + kaddr[ks];
    if constexpr (DP <= 128) asm volatile("" : "+v"(kptr[ks]));
  }
#pragma unroll
  for (int mb = 0; mb < MB; ++mb) {
    vptr[mb] = (LDS_AS const unsigned char*)smem + 2 * TILE + vaddr[mb];
    if constexpr (DP <= 128) asm volatile("" : "+v"(vptr[mb]));
  }

  f32x16 o[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[i][v] = 0.f;
  float m_run = -INFINITY, base_run = 0.f, l_run = 0.f;
  bool poison = false;  // this lane's row sees a NaN of V among its keys
  float ref = 1.17549435e-38f, ref_inv = 0.f;  // O is held in units of the largest V scale so far

  auto tile = [&](int j, auto bufc) __attribute__((always_inline)) {
    constexpr int BUF = decltype(bufc)::value;
    __syncthreads();  // tile j is in LDS; everyone is done with the other buffer
    const bool more = j + 1 < ntiles;
    // scores are in units of c0 and c1 per 32 keys; scale 0 (and a K scale of 0) must not meet the -inf of a masked score
    const float c0 = fmaxf(a.scale_log2 * sk0, 1e-30f), c1 = fmaxf(a.scale_log2 * sk1, 1e-30f);
    if (more) load_tile();
    if (wave_live && j * BN <= wave_hi) {
      f32x16 s0, s1;
#pragma unroll
      for (int v = 0; v < 16; ++v) { s0[v] = 0.f; s1[v] = 0.f; }
      {
        s16x8 ka[2][2];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          ka[ks][0] = *(LDS_AS const s16x8*)(kptr[ks] + BUF * TILE);
          ka[ks][1] = *(LDS_AS const s16x8*)(kptr[ks] + BUF * TILE + 32 * ROWB);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s0 = Mma<T>::m32(ka[ks & 1][0], qf[ks], s0);
          s1 = Mma<T>::m32(ka[ks & 1][1], qf[ks], s1);
          if (ks + 2 < KS) {
            ka[ks & 1][0] = *(LDS_AS const s16x8*)(kptr[ks + 2] + BUF * TILE);
            ka[ks & 1][1] = *(LDS_AS const s16x8*)(kptr[ks + 2] + BUF * TILE + 32 * ROWB);
          }
        }
      }
      if (j * BN + BN - 1 > wave_lo || hid0 || hid1) {
        const int lim = lim_row - j * BN - 4 * g;
        const int la = hid0 ? -1 : lim, lb = hid1 ? -1 : lim;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int e = 8 * (v >> 2) + (v & 3);
          if (e > la) s0[v] = -INFINITY;
          if (32 + e > lb) s1[v] = -INFINITY;
        }
      }
      if constexpr (F == FA_KV_E4M3) {
        if (j * BN + BN - 1 > shown && nan_tile[BUF] == j) {
#pragma clang loop unroll(disable)
          for (int v = 0; v < 32; ++v) {
            const int e = 32 * (v >> 4) + 8 * ((v & 15) >> 2) + (v & 3) + 4 * g;
            if (nan_key[BUF][e] == j && j * BN + e <= lim_row) poison = true;
          }
        }
      }
      // the compiler waits for the matrix pipe only in front of instructions it knows: the first read of each product is a
      // canonicalize, and the asm maxima depend on it
      const float g0 = __builtin_canonicalizef(s0[15]);
      float x0 = max3d(s0[0], s0[1], s0[2], g0), x1 = max3d(s0[8], s0[9], s0[10], g0);
#pragma unroll
      for (int v = 3; v < 7; v += 2) {
        x0 = max3(x0, s0[v], s0[v + 1]);
        x1 = max3(x1, s0[v + 8], s0[v + 9]);
      }
      x0 = max3(x0, s0[7], g0);
      const float g1 = __builtin_canonicalizef(s1[15]);
      float x2 = max3d(s1[0], s1[1], s1[2], g1), x3 = max3d(s1[8], s1[9], s1[10], g1);
#pragma unroll
      for (int v = 3; v < 7; v += 2) {
        x2 = max3(x2, s1[v], s1[v + 1]);
        x3 = max3(x3, s1[v + 8], s1[v + 9]);
      }
      x2 = max3(x2, s1[7], g1);
      const float mx = pair_max32(fmaxf(max2(x0, x1) * c0, max2(x2, x3) * c1));
      const bool grow = mx > m_run + kLazyLog2;
      if (__builtin_amdgcn_ballot_w64(grow) != 0) {
        const float f = grow ? fast_exp2(m_run - mx) : 1.0f;  // exp2(-inf) = 0 on the first tile
        m_run = grow ? mx : m_run;
        base_run = m_run == -INFINITY ? 0.f : m_run;
        l_run *= f;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[i][v] *= f;
      }
      const float top = fmaxf(sv0, sv1);
      if (top > ref) {  // workgroup-uniform and rare
        const float f = ref / top;
        ref = top;
        ref_inv = kLazyLift<T> / ref;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[i][v] *= f;
      }
      // The V scale of 32 keys enters as an addend of their exponents, and is divided out of their sum again: two
      // instructions instead of one for each probability.  A scale that is 0 or next to it becomes 2^-60 of the largest
      // (or 2^-67), where it cannot be seen.
      const float vf0 = fmaxf(sv0 * ref_inv, 8.67361738e-19f), vf1 = fmaxf(sv1 * ref_inv, 8.67361738e-19f);
      const float b0 = base_run - __builtin_amdgcn_logf(vf0), b1 = base_run - __builtin_amdgcn_logf(vf1);
      const float u0 = __builtin_amdgcn_rcpf(vf0), u1 = __builtin_amdgcn_rcpf(vf1);

      auto vfrag = [&](int mb, int t) {
        const s16x4 lo = lds_read_tr_lds(vptr[mb] + BUF * TILE + (16 * t) * ROWB);
        const s16x4 hi = lds_read_tr_lds(vptr[mb] + BUF * TILE + (16 * t + 8) * ROWB);
        return s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
      s16x8 va[2][MB];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) va[0][mb] = vfrag(mb, 0);
      float rs[2] = {0.f, 0.f};
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        if (t + 1 < 4) {
#pragma unroll
          for (int mb = 0; mb < MB; ++mb) va[(t + 1) & 1][mb] = vfrag(mb, t + 1);
        }
        u32x4 y;
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) {
          const int v = 8 * (t & 1) + 2 * e2;
          const float p0 = t < 2 ? fast_exp2(s0[v] * c0 - b0) : fast_exp2(s1[v] * c1 - b1);
          const float p1 = t < 2 ? fast_exp2(s0[v + 1] * c0 - b0) : fast_exp2(s1[v + 1] * c1 - b1);
          rs[t >> 1] += p0 + p1;
          y[e2] = Mma<T>::pack2(p0, p1);
        }
        const s16x8 pb = __builtin_bit_cast(s16x8, y);
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) o[mb] = Mma<T>::m32(va[t & 1][mb], pb, o[mb]);
      }
      l_run += rs[0] * u0 + rs[1] * u1;
    }
    if (more) {
      store_tile(BUF ^ 1, j + 1);
      arrived();
    }
  };

  if (ntiles > jt0) {
    store_tile(0, jt0);
    arrived();
    int j = jt0;
    for (; j + 1 < ntiles; j += 2) {
      tile(j, IC<0>{});
      tile(j + 1, IC<1>{});
    }
    if (j < ntiles) tile(j, IC<0>{});
  }

  // ---- epilogue ----
  const ArgsPtr e = args_again();
  l_run = pair_sum32(l_run);
  const int poison_other = __shfl_xor((int)poison, 32);
  const float o_unit = poison || poison_other ? __builtin_nanf("") : ref / kLazyLift<T>;
  if (e->n_splits > 1) {
    if (r < R) {
      const int64_t slot = ((rows.place + qr) * e->heads_q + hk * e->group + hg) * e->n_splits + split;
      float* dst = e->ws_o + slot * e->head_dim;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int v4 = 0; v4 < 4; ++v4) {
          const int d = 32 * mb + 8 * v4 + 4 * g;
          if (d < e->head_dim)
            *(f32x4*)(dst + d) = f32x4{o[mb][4 * v4] * o_unit, o[mb][4 * v4 + 1] * o_unit, o[mb][4 * v4 + 2] * o_unit, o[mb][4 * v4 + 3] * o_unit};
        }
      if (g == 0) *(f32x2*)(e->ws_ml + slot * 2) = f32x2{m_run, l_run};
    }
    return;
  }
  const float inv = l_run != 0.f ? o_unit / l_run : 0.f;
  __syncthreads();  // every wavefront is done with the tiles
  // whole rows go out: staged through LDS, each wavefront its own 32 rows
  constexpr int OSTR = ROWB + 16;
  unsigned char* stage = smem + wave * (32 * OSTR);
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int v4 = 0; v4 < 4; ++v4)
      *(u32x2*)(stage + c32 * OSTR + (32 * mb + 8 * v4 + 4 * g) * 2) =
          u32x2{Mma<T>::pack2(o[mb][4 * v4] * inv, o[mb][4 * v4 + 1] * inv), Mma<T>::pack2(o[mb][4 * v4 + 2] * inv, o[mb][4 * v4 + 3] * inv)};
  constexpr int RPS = 64 / CPR;
  const int sr = lane / CPR, sch = lane % CPR;
  unsigned char* ob = e->out + (e->cu_q ? 0 : (int64_t)b * e->o_sb) + (int64_t)rows.first * e->o_ss + (int64_t)hk * e->group * e->o_sh;
#pragma unroll
  for (int i = 0; i < 32 / RPS; ++i) {
    const int rl = i * RPS + sr, rr = m0 + 32 * wave + rl;
    const u32x4 x = *(const u32x4*)(stage + rl * OSTR + sch * 16);
    if (rr < R && sch * 8 < e->head_dim) {
      const int rq = rr / e->group, rh = rr - rq * e->group;
      *(u32x4*)(ob + (int64_t)rq * e->o_ss + (int64_t)rh * e->o_sh + sch * 16) = x;
    }
  }
  if (r < R && g == 0)
    e->lse[(e->cu_q ? 0 : (int64_t)b * e->lse_sb) + (int64_t)(hk * e->group + hg) * e->lse_sh + (int64_t)(rows.first + qr) * e->lse_ss] =
        l_run != 0.f ? (m_run + __builtin_log2f(l_run)) * kLn2 : INFINITY;
}

// Joins the slices of a row (a query row and head).  WPR wavefronts work on one where rows are too few to fill the chip with
// one each; RPW rows (heads of one query row) are a wavefront's where they are many, so that the loads of all of them are under
// way together.  A lane takes 4 elements of head_dim of every SPW-th slice, a load instruction 1 KiB; the first slices are
// requested before their maxima are there and before it is known whose row it is: what is left is about one memory latency.
template <typename T, int WPR, int RPW>
__global__ void __launch_bounds__(256) fa_kv_merge_kernel(const AArgs a) {
  constexpr int U = RPW == 1 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = WPR == 4 ? wave : 0;
  const int64_t r0 = WPR == 4 ? (int64_t)blockIdx.x : ((int64_t)blockIdx.x * 4 + wave) * RPW;
  if (r0 >= a.rows_q * a.heads_q) return;  // (RPW divides the heads)
  const int D = a.head_dim, ns = a.n_splits;
  const int lps = D <= 64 ? 16 : (D <= 128 ? 32 : 64), spw = 64 / lps;  // lanes a slice, slices an instruction
  const int sub = lane / lps, d = (lane % lps) * 4;
  const int s_step = WPR * spw, s_first = wr * spw + sub;
  f32x2 v[RPW];
  f32x4 x[RPW][U];
  auto load = [&](int i, int s0) {
    const float* po = a.ws_o + (r0 + i) * ns * D + min(d, D - 4);
#pragma unroll
    for (int u = 0; u < U; ++u) x[i][u] = *(const f32x4*)(po + (int64_t)min(s0 + u * s_step, ns - 1) * D);
  };
#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    v[i] = f32x2{-INFINITY, 0.f};
    if (lane < ns) v[i] = *(const f32x2*)(a.ws_ml + (r0 + i) * ns * 2 + 2 * lane);
    load(i, s_first);
  }

  const int64_t t = r0 / a.heads_q;
  const int h = (int)(r0 - t * a.heads_q);
  int b, qr, first = 0;
  if (a.cu_q) {
    ConstI32Ptr cu = (ConstI32Ptr)(uintptr_t)a.cu_q;
    int lo = 0, hi = a.batch - 1;  // the last sequence that begins at or before this row
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    b = lo;
    const QRows rows = query_rows(a.cu_q, b, a.seqlen_q, a.total_q);
    first = rows.first;
    qr = (int)t - first;
    if (qr < 0 || qr >= rows.count) return;  // (uniform over the wavefronts of the row)
  } else {
    b = (int)(t / a.seqlen_q);
    qr = (int)(t - (int64_t)b * a.seqlen_q);
  }
  unsigned char* out = a.out + (a.cu_q ? 0 : (int64_t)b * a.o_sb) + (int64_t)(first + qr) * a.o_ss + d * 2;
  float* lse = a.lse + (a.cu_q ? 0 : (int64_t)b * a.lse_sb) + (int64_t)(first + qr) * a.lse_ss;

#pragma unroll
  for (int i = 0; i < RPW; ++i) {
    float M = v[i][0];
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float f = v[i][1] == 0.f ? 0.f : fast_exp2(v[i][0] - M);  // 0: a slice without a visible key for this row
    float sum = v[i][1] * f;
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) sum += __shfl_xor(sum, o);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = s_first;;) {
      // what was loaded in the place of a slice that does not exist must not enter the sum at all, not even times 0: it may be
      // infinite
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int s = s0 + u * s_step;
        const float fs = __shfl(f, min(s, 63));
        if (s < ns) acc += x[i][u] * fs;
      }
      s0 += U * s_step;
      if (s0 - s_first >= ns) break;  // (uniform)
      load(i, s0);
    }
    for (int o = lps; o < 64; o <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
    if constexpr (WPR == 4) {
      __shared__ f32x4 part[4][64];
      part[wave][lane] = acc;
      __syncthreads();
      if (wave != 0) return;
      acc = part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane];
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    if (sub == 0 && d < D)
      *(u32x2*)(out + (int64_t)(h + i) * a.o_sh) = u32x2{Mma<T>::pack2(acc[0] * inv, acc[1] * inv), Mma<T>::pack2(acc[2] * inv, acc[3] * inv)};
    if (lane == 0) lse[(int64_t)(h + i) * a.lse_sh] = sum != 0.f ? (M + __builtin_log2f(sum)) * kLn2 : INFINITY;
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------
using namespace fa::kvhost;

template <typename T>
int launch_merge(const AArgs& a, hipStream_t st) {
  const int64_t rows = a.rows_q * a.heads_q;  // few enough for a grid, as their partial results fit the workspace
  // four wavefronts a row until one each would give every CU two workgroups; four rows a wavefront where one each
  // would go four rounds (in two slices 56480 rows 20 us against 28; in four 16000 rows 11 against 10)
  if (rows < 2048) hipLaunchKernelGGL((fa_kv_merge_kernel<T, 4, 1>), dim3((unsigned)rows), dim3(256), 0, st, a);
  else if (rows >= 32768 && a.heads_q % 4 == 0) hipLaunchKernelGGL((fa_kv_merge_kernel<T, 1, 4>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((fa_kv_merge_kernel<T, 1, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError() == hipSuccess ? FA_OK : FA_ERR_LAUNCH;
}
template <typename T, int F, int DP, int CT>
int launch_attn(const AArgs& a, int64_t wgs, hipStream_t st) {
  constexpr int NW = stream_waves(DP), lds = NW * 16 * ((DP + 4) * 4 + 8);
  constexpr auto kfn = fa_kv_attn_kernel<T, F, DP, CT, NW>;
  if (!ensure_dynamic_lds<kfn>(lds)) return FA_ERR_LAUNCH;
  hipLaunchKernelGGL(kfn, dim3((unsigned)wgs), dim3(NW * 64), lds, st, a);
  if (hipGetLastError() != hipSuccess) return FA_ERR_LAUNCH;
  return a.n_splits > 1 ? launch_merge<T>(a, st) : FA_OK;
}
template <typename T, int F, int DP>
int launch_tile(const AArgs& a, int64_t wgs, hipStream_t st) {
  constexpr int lds = 4 * 64 * DP * 2;
  constexpr auto kfn = fa_kv_tile_kernel<T, F, DP>;
  if (!ensure_dynamic_lds<kfn>(lds)) return FA_ERR_LAUNCH;
  hipLaunchKernelGGL(kfn, dim3((unsigned)wgs), dim3(256), lds, st, a);
  if (hipGetLastError() != hipSuccess) return FA_ERR_LAUNCH;
  return a.n_splits > 1 ? launch_merge<T>(a, st) : FA_OK;
}
template <typename T, int F>
int launch_attn(const AArgs& a, int tiles, int64_t wgs, hipStream_t st) {
  if (tiles == 8) return a.head_dim <= 64 ? launch_tile<T, F, 64>(a, wgs, st) : (a.head_dim <= 128 ? launch_tile<T, F, 128>(a, wgs, st) : launch_tile<T, F, 256>(a, wgs, st));
  if (a.head_dim <= 64) return tiles == 1 ? launch_attn<T, F, 64, 1>(a, wgs, st) : launch_attn<T, F, 64, 2>(a, wgs, st);
  if (a.head_dim <= 128) return tiles == 1 ? launch_attn<T, F, 128, 1>(a, wgs, st) : launch_attn<T, F, 128, 2>(a, wgs, st);
  return tiles == 1 ? launch_attn<T, F, 256, 1>(a, wgs, st) : launch_attn<T, F, 256, 2>(a, wgs, st);
}

}  // namespace

extern "C" {

int fa_kv_attn_validate(const fa_kv_attn_params* p) { return attn_validate(p); }

size_t fa_kv_attn_workspace_bytes(const fa_kv_attn_params* p) {
  return attn_validate(p) == FA_OK ? attn_workspace_bytes(p, attn_plan(p)) : 0;
}

int fa_kv_attn_launch(const fa_kv_attn_params* p, void* workspace, size_t workspace_bytes, void* stream) {
  if (const int rc = attn_validate(p)) return rc;
  const AttnPlan plan = attn_plan(p);
  const size_t need = attn_workspace_bytes(p, plan);
  if (need > 0 && (!workspace || workspace_bytes < need || misaligned(workspace, 16))) return FA_ERR_BAD_ARG;
  if (p->seqlen_q == 0 || (p->cu_seqlens_q && p->total_q == 0)) return FA_OK;
  const int64_t wgs = attn_wgs(p, plan);
  if (wgs < 0) return FA_ERR_UNSUPPORTED;
  AArgs a;
  a.q = (const unsigned char*)p->q; a.k = (const unsigned char*)p->key_pages; a.v = (const unsigned char*)p->value_pages;
  a.ks = p->key_scales; a.vs = p->value_scales;
  a.out = (unsigned char*)p->out; a.lse = p->lse;
  a.table = p->block_table; a.used = p->seqused_k; a.cu_q = p->cu_seqlens_q;
  a.q_sb = p->q_stride_b * 2; a.q_ss = p->q_stride_s * 2; a.q_sh = p->q_stride_h * 2;
  a.k_sp = p->kp_stride_p; a.k_ss = p->kp_stride_s; a.k_sh = p->kp_stride_h;
  a.v_sp = p->vp_stride_p; a.v_ss = p->vp_stride_s; a.v_sh = p->vp_stride_h;
  a.ks_sp = p->ks_stride_p; a.ks_sb = p->ks_stride_b; a.ks_sh = p->ks_stride_h;
  a.vs_sp = p->vs_stride_p; a.vs_sb = p->vs_stride_b; a.vs_sh = p->vs_stride_h;
  a.o_sb = p->o_stride_b * 2; a.o_ss = p->o_stride_s * 2; a.o_sh = p->o_stride_h * 2;
  a.lse_sb = p->lse_stride_b; a.lse_sh = p->lse_stride_h; a.lse_ss = p->lse_stride_s;
  a.bt_stride = p->block_table_stride;
  a.batch = p->batch; a.heads_q = p->heads_q; a.heads_k = p->heads_k; a.group = p->heads_q / p->heads_k;
  a.seqlen_q = p->seqlen_q; a.total_q = p->total_q; a.head_dim = p->head_dim;
  a.num_pages = p->num_pages; a.table_pages = p->table_pages; a.page_size = p->page_size;
  a.page_blocks = p->page_size / 32;
  const uint64_t sb = (uint64_t)p->scale_block / 32;  // exact: a page has at most 2^15 blocks
  a.scale_inv = (uint32_t)(((1ULL << 31) + sb - 1) / sb);
  a.is_causal = p->is_causal; a.neg_scale = p->scale < 0.f ? 1 : 0;
  a.n_splits = plan.splits; a.row_blocks = plan.row_blocks; a.hw_log2 = plan.hw_log2;
  a.scale_log2 = fabsf(p->scale) * kLog2e;
  a.ws_o = (float*)workspace;
  a.rows_q = attn_rows(p);
  a.ws_ml = a.ws_o + (need ? (size_t)a.rows_q * p->heads_q * plan.splits * p->head_dim : 0);
  hipStream_t st = (hipStream_t)stream;
  if (p->dtype == FA_DTYPE_BF16)
    return p->format == FA_KV_E4M3 ? launch_attn<__bf16, FA_KV_E4M3>(a, plan.tiles, wgs, st) : launch_attn<__bf16, FA_KV_INT8>(a, plan.tiles, wgs, st);
  return p->format == FA_KV_E4M3 ? launch_attn<_Float16, FA_KV_E4M3>(a, plan.tiles, wgs, st) : launch_attn<_Float16, FA_KV_INT8>(a, plan.tiles, wgs, st);
}

}  // extern "C"
