// ATen operators over libfa_kv.so (include/fa_kv.h, include/fa_rope.h): a serving step's plan, the paged 8-bit cache and rotary
// positions, under torch.ops.torch_mlu_amd.  The checks of what the host can see raise; work goes to the current stream of the
// tensors' device.
#include <ATen/ATen.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>
#include <limits>
#include <tuple>

#include "fa_kv.h"
#include "fa_rope.h"

namespace torch_mlu_amd {
namespace {

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

void check_rc(const char* what, int rc) { TORCH_CHECK(rc == FA_OK, what, " failed: ", fa_kv_error_string(rc), " (rc=", rc, ")"); }

// a small int32 tensor of the device that the others are on
void check_ints(const at::Tensor& t, const char* name, int64_t dim, const at::Device& dev) {
  TORCH_CHECK(t.device() == dev, name, " must be on ", dev, ", got ", t.device());
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must have dtype int32");
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimension", dim == 1 ? "" : "s");
  if (t.numel() > 0) TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, " must have contiguous rows");
}

int32_t narrow(int64_t x, const char* name) {
  TORCH_CHECK(x >= 0 && x <= std::numeric_limits<int32_t>::max(), name, " is out of range: ", x);
  return static_cast<int32_t>(x);
}

// stride of a dimension; one of a single entry is never used and may be anything
int64_t dim_stride(const at::Tensor& t, int64_t d) { return t.size(d) > 1 ? t.stride(d) : 0; }

void check_inference(const at::Tensor& t, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what, " is for inference: it has no gradient");
}

// ---- pages and scales, as write and attention take them ---------------------------------------------------------------
template <typename P>
void fill_pool(P& p, const at::Tensor& kp, const at::Tensor& vp, const at::Tensor& ks, const at::Tensor& vs, int64_t heads, int64_t head_dim,
               const at::Device& dev) {
  const at::Tensor* pages[] = {&kp, &vp};
  const at::Tensor* scales[] = {&ks, &vs};
  const char* pname[] = {"key_pages", "value_pages"};
  const char* sname[] = {"key_scales", "value_scales"};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = *pages[i];
    TORCH_CHECK(t.device() == dev, pname[i], " must be on ", dev, ", got ", t.device());
    TORCH_CHECK(t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kChar, pname[i], " must have dtype float8_e4m3fn or int8, got ",
                t.scalar_type());
    check_inference(t, pname[i]);
    TORCH_CHECK(t.dim() == 4, pname[i], " must be [pages, page_size, heads, head_dim]");
    TORCH_CHECK(t.size(2) == heads && t.size(3) == head_dim, pname[i], " must have ", heads, " heads of ", head_dim, ", got ", t.sizes());
    TORCH_CHECK(t.size(3) <= 1 || t.stride(3) == 1, pname[i], " must have a contiguous last dimension");
    const at::Tensor& s = *scales[i];
    TORCH_CHECK(s.device() == dev, sname[i], " must be on ", dev, ", got ", s.device());
    TORCH_CHECK(s.scalar_type() == at::kFloat, sname[i], " must have dtype float32");
    check_inference(s, sname[i]);
    TORCH_CHECK(s.dim() == 3 && s.size(0) == t.size(0) && s.size(2) == heads, sname[i], " must be [pages, blocks, heads], got ", s.sizes());
  }
  TORCH_CHECK(kp.scalar_type() == vp.scalar_type() && kp.sizes() == vp.sizes(), "key_pages and value_pages must have the same dtype and shape");
  TORCH_CHECK(ks.sizes() == vs.sizes(), "key_scales and value_scales must have the same shape");
  const int64_t page_size = kp.size(1), blocks = ks.size(1);
  TORCH_CHECK(kp.size(0) > 0 && page_size > 0, "the cache has no pages");
  TORCH_CHECK(blocks > 0 && page_size % blocks == 0 && page_size / blocks % 32 == 0,
              "a page must have whole blocks of a multiple of 32 tokens, one scale each: page_size ", page_size, ", ", blocks, " scales");
  TORCH_CHECK(head_dim >= 16 && head_dim <= 256 && head_dim % 16 == 0, "head_dim must be a multiple of 16, at most 256, got ", head_dim);
  p.key_pages = kp.data_ptr();
  p.value_pages = vp.data_ptr();
  p.key_scales = ks.data_ptr<float>();
  p.value_scales = vs.data_ptr<float>();
  p.kp_stride_p = dim_stride(kp, 0); p.kp_stride_s = dim_stride(kp, 1); p.kp_stride_h = dim_stride(kp, 2);
  p.vp_stride_p = dim_stride(vp, 0); p.vp_stride_s = dim_stride(vp, 1); p.vp_stride_h = dim_stride(vp, 2);
  p.ks_stride_p = dim_stride(ks, 0); p.ks_stride_b = dim_stride(ks, 1); p.ks_stride_h = dim_stride(ks, 2);
  p.vs_stride_p = dim_stride(vs, 0); p.vs_stride_b = dim_stride(vs, 1); p.vs_stride_h = dim_stride(vs, 2);
  p.head_dim = static_cast<int32_t>(head_dim);
  p.num_pages = narrow(kp.size(0), "the number of pages");
  p.page_size = narrow(page_size, "page_size");
  p.scale_block = narrow(page_size / blocks, "the block of a scale");
  p.format = kp.scalar_type() == at::kChar ? FA_KV_INT8 : FA_KV_E4M3;
}

int dtype_16(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, name, " must have dtype float16 or bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_FP16;
}

// rows that 16-byte accesses can take, or a copy
at::Tensor aligned_rows(const at::Tensor& t) {
  bool ok = t.size(-1) <= 1 || t.stride(-1) == 1;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && dim_stride(t, d) % 8 == 0;
  ok = ok && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

// A contiguous tensor in a part of `bytes`, which keeps the whole of it alive.  (Six small allocations cost twice the kernel.)
at::Tensor part_of(const at::Tensor& bytes, int64_t& at_byte, at::ScalarType dtype, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(bytes.storage()), bytes.key_set(), c10::scalarTypeToTypeMeta(dtype));
  const int64_t size = static_cast<int64_t>(c10::elementSize(dtype));
  impl->set_storage_offset(at_byte / size);
  impl->set_sizes_contiguous({n});
  at_byte += n * size;
  return at::Tensor(std::move(impl));
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> paged_plan(
    const at::Tensor& cached, const at::Tensor& new_tokens, const at::Tensor& block_table, const at::Tensor& free_pages, const at::Tensor& free_count,
    int64_t page_size, int64_t max_tokens) {
  TORCH_CHECK(cached.is_cuda(), "Input tensor must be on HIP device");
  const auto dev = cached.device();
  check_ints(cached, "cached", 1, dev);
  check_ints(new_tokens, "new_tokens", 1, dev);
  check_ints(block_table, "block_table", 2, dev);
  check_ints(free_pages, "free_pages", 1, dev);
  check_ints(free_count, "free_count", 1, dev);
  TORCH_CHECK(free_count.numel() == 1, "free_count must have one entry");
  const int64_t B = cached.size(0);
  TORCH_CHECK(new_tokens.size(0) == B && block_table.size(0) == B, "cached, new_tokens and block_table must have one entry for each request");
  TORCH_CHECK(B <= FA_KV_MAX_BATCH, "at most ", FA_KV_MAX_BATCH, " requests, got ", B);
  TORCH_CHECK(page_size > 0, "page_size must be positive");
  TORCH_CHECK(max_tokens >= 0, "max_tokens must not be negative");
  narrow(max_tokens, "max_tokens");
  const c10::OptionalDeviceGuard guard(dev);
  const at::Tensor bytes = at::empty({max_tokens * 12 + (2 * B + 2) * 4 + B}, cached.options().dtype(at::kByte));
  int64_t used_bytes = 0;
  at::Tensor slots = part_of(bytes, used_bytes, at::kLong, max_tokens), positions = part_of(bytes, used_bytes, at::kInt, max_tokens);
  at::Tensor cu = part_of(bytes, used_bytes, at::kInt, B + 1), used = part_of(bytes, used_bytes, at::kInt, B);
  at::Tensor left = part_of(bytes, used_bytes, at::kInt, 1), admitted = part_of(bytes, used_bytes, at::kBool, B);
  fa_kv_plan_params p{};
  p.cached = cached.data_ptr<int32_t>();
  p.new_tokens = new_tokens.data_ptr<int32_t>();
  p.block_table = block_table.data_ptr<int32_t>();
  p.free_pages = free_pages.data_ptr<int32_t>();
  p.free_count = free_count.data_ptr<int32_t>();
  p.cu_seqlens = cu.data_ptr<int32_t>();
  p.seqused = used.data_ptr<int32_t>();
  p.positions = positions.data_ptr<int32_t>();
  p.slots = slots.data_ptr<int64_t>();
  p.admitted = static_cast<uint8_t*>(admitted.data_ptr());
  p.free_left = left.data_ptr<int32_t>();
  p.block_table_stride = B > 1 ? block_table.stride(0) : block_table.size(1);
  p.batch = static_cast<int32_t>(B);
  p.table_pages = narrow(block_table.size(1), "the width of block_table");
  p.page_size = narrow(page_size, "page_size");
  p.max_tokens = narrow(max_tokens, "max_tokens");
  p.free_capacity = narrow(free_pages.size(0), "the length of free_pages");
  check_rc("paged_plan", fa_kv_plan_launch(&p, stream_of(cached)));
  return {cu, used, positions, slots, admitted, left};
}

void paged_cache_write(const at::Tensor& key, const at::Tensor& value, const at::Tensor& key_pages, const at::Tensor& value_pages,
                       const at::Tensor& key_scales, const at::Tensor& value_scales, const at::Tensor& slots) {
  TORCH_CHECK(key.is_cuda(), "Input tensor must be on HIP device");
  const auto dev = key.device();
  TORCH_CHECK(key.dim() == 3 && value.dim() == 3 && key.sizes() == value.sizes(), "key and value must be [tokens, heads, head_dim], got ", key.sizes(),
              " and ", value.sizes());
  TORCH_CHECK(value.device() == dev, "value must be on ", dev, ", got ", value.device());
  TORCH_CHECK(value.scalar_type() == key.scalar_type(), "key and value must have the same dtype");
  TORCH_CHECK(slots.device() == dev, "slots must be on ", dev, ", got ", slots.device());
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.size(0) == key.size(0), "slots must be int64 [tokens]");
  TORCH_CHECK(slots.size(0) <= 1 || slots.stride(0) == 1, "slots must be contiguous");
  check_inference(key, "paged_cache_write");
  check_inference(value, "paged_cache_write");
  fa_kv_write_params p{};
  p.dtype = dtype_16(key, "key");
  const c10::OptionalDeviceGuard guard(dev);
  fill_pool(p, key_pages, value_pages, key_scales, value_scales, key.size(1), key.size(2), dev);
  if (key.size(0) == 0) return;
  const at::Tensor k = aligned_rows(key), v = aligned_rows(value);
  p.key = k.data_ptr();
  p.value = v.data_ptr();
  p.slots = slots.data_ptr<int64_t>();
  p.key_stride_t = dim_stride(k, 0); p.key_stride_h = dim_stride(k, 1);
  p.value_stride_t = dim_stride(v, 0); p.value_stride_h = dim_stride(v, 1);
  p.tokens = narrow(k.size(0), "the number of tokens");
  p.heads = narrow(k.size(1), "the number of heads");
  check_rc("paged_cache_write", fa_kv_write_launch(&p, stream_of(key)));
}

std::tuple<at::Tensor, at::Tensor> paged_attention_8bit(const at::Tensor& query, const at::Tensor& key_pages, const at::Tensor& value_pages,
                                                        const at::Tensor& key_scales, const at::Tensor& value_scales, const at::Tensor& block_table,
                                                        const at::Tensor& seqused_k, const std::optional<at::Tensor>& cu_seqlens_q,
                                                        std::optional<int64_t> max_seqlen_q, bool is_causal, std::optional<double> scale) {
  TORCH_CHECK(query.is_cuda(), "Input tensor must be on HIP device");
  const auto dev = query.device();
  const bool packed = cu_seqlens_q.has_value();
  TORCH_CHECK(query.dim() == (packed ? 3 : 4), packed ? "query must be [tokens, heads, head_dim] with cu_seqlens_q" : "query must be [batch, heads, rows, head_dim]",
              ", got ", query.sizes());
  check_inference(query, "paged_attention");
  fa_kv_attn_params p{};
  p.dtype = dtype_16(query, "query");
  check_ints(block_table, "block_table", 2, dev);
  check_ints(seqused_k, "seqused_k", 1, dev);
  const int64_t Hq = query.size(1), D = query.size(-1);
  int64_t B, Sq;
  if (packed) {
    check_ints(*cu_seqlens_q, "cu_seqlens_q", 1, dev);
    TORCH_CHECK(cu_seqlens_q->numel() >= 1, "cu_seqlens_q must have batch + 1 entries");
    TORCH_CHECK(max_seqlen_q.has_value() && *max_seqlen_q >= 0, "cu_seqlens_q needs max_seqlen_q");
    B = cu_seqlens_q->numel() - 1;
    Sq = std::min(*max_seqlen_q, query.size(0));
  } else {
    TORCH_CHECK(!max_seqlen_q.has_value(), "max_seqlen_q goes with cu_seqlens_q");
    B = query.size(0);
    Sq = query.size(2);
  }
  TORCH_CHECK(block_table.size(0) == B && seqused_k.size(0) == B, "block_table and seqused_k must have one entry for each of ", B, " sequences");
  TORCH_CHECK(key_pages.dim() == 4, "key_pages must be [pages, page_size, heads, head_dim]");
  const int64_t Hk = key_pages.size(2);
  TORCH_CHECK(Hk > 0 && Hq % Hk == 0, "the number of heads in key_pages must divide that in query: ", Hk, " and ", Hq);
  const c10::OptionalDeviceGuard guard(dev);
  fill_pool(p, key_pages, value_pages, key_scales, value_scales, Hk, D, dev);
  const at::Tensor q = aligned_rows(query);
  const auto floats = query.options().dtype(at::kFloat);
  at::Tensor out, lse;
  if (packed) {
    // rows that no sequence owns stay what they are here
    out = at::empty({q.size(0), Hq, D}, query.options());
    lse = at::empty({Hq, q.size(0)}, floats);
    p.q_stride_s = dim_stride(q, 0); p.q_stride_h = dim_stride(q, 1);
    p.o_stride_s = out.stride(0); p.o_stride_h = out.stride(1);
    p.lse_stride_h = lse.stride(0); p.lse_stride_s = lse.stride(1);
    p.cu_seqlens_q = cu_seqlens_q->data_ptr<int32_t>();
    p.total_q = narrow(q.size(0), "the number of rows");
  } else {
    out = at::empty_strided({B, Hq, Sq, D}, {Sq * Hq * D, D, Hq * D, 1}, query.options());  // [B, Sq, Hq, D] in memory
    lse = at::empty({B, Hq, Sq}, floats);
    p.q_stride_b = dim_stride(q, 0); p.q_stride_h = dim_stride(q, 1); p.q_stride_s = dim_stride(q, 2);
    p.o_stride_b = out.stride(0); p.o_stride_h = out.stride(1); p.o_stride_s = out.stride(2);
    p.lse_stride_b = lse.stride(0); p.lse_stride_h = lse.stride(1); p.lse_stride_s = lse.stride(2);
  }
  if (out.numel() == 0 || B == 0) return {out, lse};
  p.q = q.data_ptr();
  p.out = out.data_ptr();
  p.lse = lse.data_ptr<float>();
  p.block_table = block_table.data_ptr<int32_t>();
  p.seqused_k = seqused_k.data_ptr<int32_t>();
  p.block_table_stride = B > 1 ? block_table.stride(0) : block_table.size(1);
  p.batch = narrow(B, "the batch");
  p.heads_q = narrow(Hq, "the number of heads");
  p.heads_k = narrow(Hk, "the number of heads");
  p.seqlen_q = narrow(Sq, "the number of rows");
  p.table_pages = narrow(block_table.size(1), "the width of block_table");
  p.scale = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(D)));
  p.is_causal = is_causal ? 1 : 0;
  if (block_table.size(1) == 0) {  // no keys at all
    out.zero_();
    lse.fill_(std::numeric_limits<float>::infinity());
    return {out, lse};
  }
  const size_t need = fa_kv_attn_workspace_bytes(&p);
  at::Tensor ws;
  if (need) ws = at::empty({static_cast<int64_t>(need)}, query.options().dtype(at::kByte));
  check_rc("paged_attention", fa_kv_attn_launch(&p, need ? ws.data_ptr() : nullptr, need, stream_of(query)));
  return {out, lse};
}

// ---- rotary positions -----------------------------------------------------------------------------------------------------
namespace {

std::tuple<at::Tensor, at::Tensor> rotary_forward(const at::Tensor& query, const at::Tensor& key, const at::Tensor& positions, const at::Tensor& inv_freq,
                                                  const at::Tensor& axes, bool interleaved, bool inverse) {
  const auto dev = query.device();
  const c10::OptionalDeviceGuard guard(dev);
  const bool packed = query.dim() == 3;
  fa_rope_params p{};
  const auto t = query.scalar_type();
  p.dtype = t == at::kFloat ? FA_DTYPE_FP32 : (t == at::kBFloat16 ? FA_DTYPE_BF16 : FA_DTYPE_FP16);
  p.batch = narrow(packed ? 1 : query.size(0), "the batch");
  p.seqlen = narrow(packed ? query.size(0) : query.size(2), "the number of tokens");
  p.heads_q = narrow(query.size(1), "the number of heads");
  p.heads_k = key.defined() ? narrow(key.size(1), "the number of heads") : 0;
  p.head_dim = narrow(query.size(-1), "head_dim");
  p.pairs = narrow(inv_freq.size(0), "the number of frequencies");
  p.num_axes = narrow(positions.size(0), "the number of axes");
  p.positions_64 = positions.scalar_type() == at::kLong;
  p.inv_freq_64 = inv_freq.scalar_type() == at::kDouble;
  p.interleaved = interleaved;
  p.inverse = inverse;
  const at::Tensor freq = inv_freq.contiguous(), ax = axes.contiguous();
  p.positions = positions.data_ptr();
  p.inv_freq = freq.data_ptr();
  p.axes = ax.data_ptr<int32_t>();
  p.pos_stride_a = positions.stride(0);
  p.pos_stride_b = positions.dim() == 3 ? positions.stride(1) : 0;
  p.pos_stride_s = positions.stride(-1);
  at::Tensor x[2], y[2];
  const at::Tensor* in[2] = {&query, &key};
  for (int i = 0; i < 2; ++i) {
    if (!in[i]->defined()) continue;
    x[i] = in[i]->size(-1) > 1 && in[i]->stride(-1) != 1 ? in[i]->contiguous() : *in[i];
    y[i] = at::empty_like(x[i]);
    if (y[i].size(-1) > 1 && y[i].stride(-1) != 1) y[i] = at::empty(x[i].sizes(), x[i].options());
  }
  const int s = packed ? 0 : 2;
  p.q = x[0].data_ptr(); p.q_out = y[0].data_ptr();
  p.q_stride_b = packed ? 0 : dim_stride(x[0], 0); p.q_stride_s = dim_stride(x[0], s); p.q_stride_h = dim_stride(x[0], 1);
  p.qo_stride_b = packed ? 0 : dim_stride(y[0], 0); p.qo_stride_s = dim_stride(y[0], s); p.qo_stride_h = dim_stride(y[0], 1);
  if (key.defined()) {
    p.k = x[1].data_ptr(); p.k_out = y[1].data_ptr();
    p.k_stride_b = packed ? 0 : dim_stride(x[1], 0); p.k_stride_s = dim_stride(x[1], s); p.k_stride_h = dim_stride(x[1], 1);
    p.ko_stride_b = packed ? 0 : dim_stride(y[1], 0); p.ko_stride_s = dim_stride(y[1], s); p.ko_stride_h = dim_stride(y[1], 1);
  }
  if (query.numel() > 0 || (key.defined() && key.numel() > 0)) check_rc("rotary", fa_rope_launch(&p, stream_of(query)));
  return {y[0], y[1]};
}

void check_rotary(const at::Tensor& query, const at::Tensor& key, const at::Tensor& positions, const at::Tensor& inv_freq, const at::Tensor& axes) {
  TORCH_CHECK(query.is_cuda(), "Input tensor must be on HIP device");
  const auto dev = query.device();
  const auto t = query.scalar_type();
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, "query must have dtype float32, float16 or bfloat16, got ", t);
  TORCH_CHECK(query.dim() == 3 || query.dim() == 4, "query must be [batch, heads, rows, head_dim] or packed [tokens, heads, head_dim], got ", query.sizes());
  const bool packed = query.dim() == 3;
  TORCH_CHECK(query.size(1) > 0, "query has no heads");
  if (key.defined()) {
    TORCH_CHECK(key.device() == dev, "key must be on ", dev, ", got ", key.device());
    TORCH_CHECK(key.scalar_type() == t, "query and key must have the same dtype");
    TORCH_CHECK(key.dim() == query.dim() && key.size(-1) == query.size(-1) && key.size(0) == query.size(0) && (packed || key.size(2) == query.size(2)),
                "query and key must have the same tokens and head_dim, got ", query.sizes(), " and ", key.sizes());
  }
  TORCH_CHECK(positions.device() == dev, "positions must be on ", dev, ", got ", positions.device());
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, "positions must have dtype int32 or int64");
  const bool shaped = packed ? positions.dim() == 2 && positions.size(1) == query.size(0)
                             : (positions.dim() == 2 && positions.size(1) == query.size(2)) ||
                                   (positions.dim() == 3 && positions.size(1) == query.size(0) && positions.size(2) == query.size(2));
  TORCH_CHECK(shaped, "positions must be [axes, ", packed ? "tokens]" : "rows] or [axes, batch, rows]", ", got ", positions.sizes());
  TORCH_CHECK(positions.size(0) >= 1 && positions.size(0) <= FA_ROPE_MAX_AXES, "1 to ", FA_ROPE_MAX_AXES, " axes, got ", positions.size(0));
  TORCH_CHECK(inv_freq.device() == dev && axes.device() == dev, "inv_freq and axes must be on ", dev);
  TORCH_CHECK(inv_freq.scalar_type() == at::kDouble || inv_freq.scalar_type() == at::kFloat, "inv_freq must have dtype float64 or float32");
  TORCH_CHECK(axes.scalar_type() == at::kInt, "axes must have dtype int32");
  TORCH_CHECK(inv_freq.dim() == 1 && axes.sizes() == inv_freq.sizes(), "inv_freq and axes must have one entry for each pair");
  TORCH_CHECK(inv_freq.size(0) >= 1 && 2 * inv_freq.size(0) <= query.size(-1), "1 to head_dim / 2 pairs, got ", inv_freq.size(0), " for a head_dim of ",
              query.size(-1));
  TORCH_CHECK(query.size(-1) <= 512, "head_dim at most 512, got ", query.size(-1));
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> rotary(const at::Tensor& query, const std::optional<at::Tensor>& key, const at::Tensor& positions,
                                          const at::Tensor& inv_freq, const at::Tensor& axes, bool interleaved, bool inverse);

namespace {

struct Rotary : public torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& query,
                                                const std::optional<at::Tensor>& optional_key, const at::Tensor& positions,
                                                const at::Tensor& inv_freq, const at::Tensor& axes, bool interleaved, bool inverse) {
    at::AutoDispatchBelowADInplaceOrView below;
    const at::Tensor key = optional_key.value_or(at::Tensor());
    auto [q, k] = rotary_forward(query, key, positions, inv_freq, axes, interleaved, inverse);
    ctx->save_for_backward({positions, inv_freq, axes});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->set_materialize_grads(false);
    torch::autograd::variable_list fixed;
    if (!query.requires_grad()) fixed.push_back(q);
    if (key.defined() && !key.requires_grad()) fixed.push_back(k);
    ctx->mark_non_differentiable(fixed);
    if (!key.defined()) return {q};
    return {q, k};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
    at::Tensor gq = grads[0], gk = grads.size() > 1 ? grads[1] : at::Tensor();
    at::Tensor dq, dk;
    if (gq.defined()) {
      std::tie(dq, dk) = rotary(gq, gk.defined() ? std::optional<at::Tensor>(gk) : std::nullopt, saved[0], saved[1], saved[2], interleaved, !inverse);
      if (!gk.defined()) dk = at::Tensor();
    } else if (gk.defined()) {
      dk = std::get<0>(rotary(gk, std::nullopt, saved[0], saved[1], saved[2], interleaved, !inverse));
    }
    return {dq, dk, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

std::tuple<at::Tensor, at::Tensor> rotary(const at::Tensor& query, const std::optional<at::Tensor>& key, const at::Tensor& positions,
                                          const at::Tensor& inv_freq, const at::Tensor& axes, bool interleaved, bool inverse) {
  const at::Tensor k = key.has_value() ? *key : at::Tensor();
  check_rotary(query, k, positions, inv_freq, axes);
  std::tuple<at::Tensor, at::Tensor> r;
  if (at::GradMode::is_enabled() && (query.requires_grad() || (k.defined() && k.requires_grad()))) {
    const auto y = Rotary::apply(query, key, positions, inv_freq, axes, interleaved, inverse);
    r = {y[0], k.defined() ? y[1] : at::Tensor()};
  } else {
    r = rotary_forward(query, k, positions, inv_freq, axes, interleaved, inverse);
  }
  if (!k.defined()) std::get<1>(r) = at::empty({0}, query.options());
  return r;
}

}  // namespace torch_mlu_amd

TORCH_LIBRARY_FRAGMENT(torch_mlu_amd, m) {
  m.def("paged_plan(Tensor cached, Tensor new_tokens, Tensor(a!) block_table, Tensor free_pages, Tensor free_count, int page_size, int max_tokens) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        &torch_mlu_amd::paged_plan);
  m.def("paged_cache_write(Tensor key, Tensor value, Tensor(a!) key_pages, Tensor(b!) value_pages, Tensor(c!) key_scales, Tensor(d!) value_scales, "
        "Tensor slots) -> ()",
        &torch_mlu_amd::paged_cache_write);
  m.def("paged_attention_8bit(Tensor query, Tensor key_pages, Tensor value_pages, Tensor key_scales, Tensor value_scales, Tensor block_table, "
        "Tensor seqused_k, Tensor? cu_seqlens_q, int? max_seqlen_q, bool is_causal, float? scale) -> (Tensor, Tensor)",
        &torch_mlu_amd::paged_attention_8bit);
  m.def("rotary(Tensor query, Tensor? key, Tensor positions, Tensor inv_freq, Tensor axes, bool interleaved, bool inverse) -> (Tensor, Tensor)",
        &torch_mlu_amd::rotary);
}
