// functs:: operators of a paged key / value cache held in 8 bits (fx_kv_* of include/fxhip.h): what a program
// of attention over growing caches (functs/benchmark/simpleops/attention/attention.py:38-58) calls when it serves
// many requests of different lengths.
//   functs::kv_plan       pages, slots and offsets of a step's tokens, from lengths on the device
//   functs::kv_store      writes keys and values
//   functs::kv_read       gives them back as numbers
//   functs::kv_attention  attention over them
// Nothing here waits for the device or reads from it: a captured call serves other lengths when it is replayed.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>

#include "../../../include/fxhip.h"

namespace functs {
namespace {
using at::Tensor;

#define FX_OK_OR_THROW(expr)                                             \
  do {                                                                   \
    int rc__ = (expr);                                                   \
    TORCH_CHECK(rc__ >= 0, "fxhip: ", fx_last_error(), " (", #expr, ")"); \
  } while (0)

void* streamOf(c10::Device dev) { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream(); }
// (tensors made in inference mode carry no version)
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void onGpu(const char* op, const Tensor& t, const char* name, c10::Device dev) {
  TORCH_CHECK(t.is_cuda(), op, " runs on the GPU only; ", name, " is a ", t.device(), " tensor");
  TORCH_CHECK(t.device() == dev, op, ": ", name, " is on ", t.device(), ", the others on ", dev);
}
void noGrad(const char* op, const Tensor& t, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), op, " has no backward pass: ", name, " requires a gradient");
  TORCH_CHECK(!t._fw_grad(0).defined(), op, " has no derivative: ", name, " carries a tangent");
}
int32_t sized(const char* op, int64_t n, const char* name) {
  TORCH_CHECK(n >= 0 && n <= INT32_MAX, op, ": ", name, " is out of range (", n, ")");
  return (int32_t)n;
}
Tensor ints(const char* op, const Tensor& t, const char* name, int64_t n, c10::Device dev) {
  onGpu(op, t, name, dev);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && (n < 0 || t.size(0) == n), op, ": ", name, " must be int32 [", n < 0 ? t.numel() : n,
              "], got ", t.scalar_type(), " ", t.sizes());
  return t.contiguous();
}
int dtypeOf(const char* op, at::ScalarType t, const char* name) {
  TORCH_CHECK(t == at::kFloat || t == at::kHalf || t == at::kBFloat16, op, ": ", name, " must be float32, float16 or bfloat16, got ", t);
  return t == at::kFloat ? FX_DT_F32 : t == at::kHalf ? FX_DT_F16 : FX_DT_BF16;
}

// [pages, heads, page, depth] codes; a page's codes lie side by side, pages anywhere
fx_kv_cache cacheOf(const char* op, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  TORCH_CHECK(k.dim() == 4, op, ": k_cache must be [pages, heads, page, depth], got ", k.sizes());
  TORCH_CHECK(k.size(0) >= 1 && k.size(1) >= 1, op, ": a cache has at least one page and one head, got ", k.sizes());
  TORCH_CHECK(k.is_cuda(), op, " runs on the GPU only; k_cache is a ", k.device(), " tensor");
  const auto dev = k.device();
  onGpu(op, v, "v_cache", dev);
  onGpu(op, ks, "k_scale", dev);
  onGpu(op, vs, "v_scale", dev);
  noGrad(op, k, "k_cache");
  noGrad(op, v, "v_cache");
  noGrad(op, ks, "k_scale");
  noGrad(op, vs, "v_scale");
  TORCH_CHECK(k.scalar_type() == at::kFloat8_e4m3fn || k.scalar_type() == at::kChar, op, ": a cache holds float8_e4m3fn or int8, got ", k.scalar_type());
  const int64_t N = k.size(0), H = k.size(1), P = k.size(2), D = k.size(3);
  TORCH_CHECK(v.scalar_type() == k.scalar_type() && v.dim() == 5 && v.size(0) == N && v.size(1) == H && v.size(2) * 16 == P && v.size(3) == D && v.size(4) == 16,
              op, ": v_cache must be [pages, heads, page / 16, depth, 16] of the type of k_cache, got ", v.scalar_type(), " ", v.sizes(), " beside ", k.sizes());
  for (const Tensor* s : {&ks, &vs})
    TORCH_CHECK(s->scalar_type() == at::kFloat && s->dim() == 2 && s->size(0) == N && s->size(1) == H && (H == 1 || s->stride(1) == 1), op,
                ": scales must be float32 [pages, heads], heads side by side, got ", s->scalar_type(), " ", s->sizes());
  const auto packed = [](const Tensor& t) {   // (sizes of 1 have any stride)
    int64_t step = 1;
    for (int64_t d = t.dim() - 1; d > 0; step *= t.size(d--))
      if (t.size(d) != 1 && t.stride(d) != step) return false;
    return true;
  };
  TORCH_CHECK(packed(k) && packed(v), op, ": a page of the cache must be contiguous");
  fx_kv_cache c;
  memset(&c, 0, sizeof c);
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.k_scale = ks.data_ptr<float>();
  c.v_scale = vs.data_ptr<float>();
  c.k_page_stride = k.stride(0);
  c.v_page_stride = v.stride(0);
  c.k_scale_page_stride = ks.stride(0);
  c.v_scale_page_stride = vs.stride(0);
  c.pages = sized(op, N, "the number of pages");
  c.heads = sized(op, H, "the number of heads");
  c.page_size = sized(op, P, "the page size");
  c.depth = sized(op, D, "the depth");
  c.held = k.scalar_type() == at::kChar ? FX_KV_INT8 : FX_KV_E4M3;
  return c;
}

Tensor slotsOf(const char* op, const Tensor& slots, c10::Device dev) {
  onGpu(op, slots, "slots", dev);
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 1, op, ": slots must be int64 [tokens], got ", slots.scalar_type(), " ", slots.sizes());
  return slots.contiguous();
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> kvPlan(const Tensor& past_lens, const Tensor& new_lens, Tensor block_table, const Tensor& free_pages,
                                                          int64_t page_size, int64_t max_tokens, const std::optional<Tensor>& free_start) {
  static const char op[] = "functs::kv_plan";
  TORCH_CHECK(block_table.is_cuda(), op, " runs on the GPU only; block_table is a ", block_table.device(), " tensor");
  const auto dev = block_table.device();
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && (block_table.size(1) <= 1 || block_table.stride(1) == 1), op,
              ": block_table must be int32 [requests, columns], columns side by side, got ", block_table.scalar_type(), " ", block_table.sizes());
  const int64_t B = block_table.size(0);
  const Tensor past = ints(op, past_lens, "past_lens", B, dev), added = ints(op, new_lens, "new_lens", B, dev), pages = ints(op, free_pages, "free_pages", -1, dev);
  Tensor from;
  if (free_start && free_start->defined()) {
    onGpu(op, *free_start, "free_start", dev);
    TORCH_CHECK(free_start->scalar_type() == at::kInt && free_start->numel() == 1, op, ": free_start must be one int32");
    from = *free_start;
  }
  c10::DeviceGuard guard(dev);
  const auto i32 = at::TensorOptions().dtype(at::kInt).device(dev);
  fx_kv_plan_desc d;
  memset(&d, 0, sizeof d);
  d.tokens = sized(op, max_tokens, "max_tokens");
  d.requests = sized(op, B, "the number of requests");
  d.columns = sized(op, block_table.size(1), "the number of columns");
  d.n_free = sized(op, pages.numel(), "the number of free pages");
  TORCH_CHECK(page_size >= 16 && page_size <= 256, op, ": page_size must be 16, 32, 64, 128 or 256, got ", page_size);
  d.page_size = (int32_t)page_size;
  Tensor slots = at::empty({max_tokens}, i32.dtype(at::kLong)), positions = at::empty({max_tokens}, i32), starts = at::empty({B + 1}, i32),
         lens = at::empty({B}, i32), taken = at::empty({1}, i32);
  d.past = past.data_ptr<int32_t>();
  d.added = added.data_ptr<int32_t>();
  d.free_pages = pages.data_ptr<int32_t>();
  d.free_start = from.defined() ? from.data_ptr<int32_t>() : nullptr;
  d.table = block_table.data_ptr<int32_t>();
  d.table_stride = block_table.stride(0);
  d.slots = slots.data_ptr<int64_t>();
  d.positions = positions.data_ptr<int32_t>();
  d.starts = starts.data_ptr<int32_t>();
  d.lens = lens.data_ptr<int32_t>();
  d.taken = taken.data_ptr<int32_t>();
  FX_OK_OR_THROW(fx_kv_plan(&d, streamOf(dev)));
  written(block_table);
  return {slots, positions, starts, lens, taken};
}

// rows [tokens, heads, depth], a depth contiguous
void rowsOf(const char* op, const Tensor& t, const char* name, const fx_kv_cache& c, int64_t tokens, c10::Device dev) {
  onGpu(op, t, name, dev);
  TORCH_CHECK(t.dim() == 3 && t.size(0) == tokens && t.size(1) == c.heads && t.size(2) == c.depth, op, ": ", name, " must be [", tokens, ", ", c.heads, ", ",
              c.depth, "], got ", t.sizes());
}
fx_kv_rows rowsDesc(const Tensor& k, const Tensor& v, const Tensor& slots, int32_t tokens, int dtype) {
  fx_kv_rows r;
  memset(&r, 0, sizeof r);
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  r.k_token_stride = k.stride(0);
  r.k_head_stride = k.stride(1);
  r.v_token_stride = v.stride(0);
  r.v_head_stride = v.stride(1);
  r.slots = slots.data_ptr<int64_t>();
  r.tokens = tokens;
  r.dtype = dtype;
  return r;
}

void kvStore(const Tensor& k_, const Tensor& v_, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, const Tensor& slots_) {
  static const char op[] = "functs::kv_store";
  const fx_kv_cache c = cacheOf(op, k_cache, v_cache, k_scale, v_scale);
  const auto dev = k_cache.device();
  const Tensor slots = slotsOf(op, slots_, dev);
  const int32_t tokens = sized(op, slots.numel(), "the number of tokens");
  rowsOf(op, k_, "k", c, tokens, dev);
  rowsOf(op, v_, "v", c, tokens, dev);
  noGrad(op, k_, "k");
  noGrad(op, v_, "v");
  TORCH_CHECK(k_.scalar_type() == v_.scalar_type(), op, ": k and v must be of one type, got ", k_.scalar_type(), " and ", v_.scalar_type());
  const int dtype = dtypeOf(op, k_.scalar_type(), "k");
  c10::DeviceGuard guard(dev);
  const Tensor k = k_.stride(2) == 1 ? k_ : k_.contiguous(), v = v_.stride(2) == 1 ? v_ : v_.contiguous();
  const fx_kv_rows r = rowsDesc(k, v, slots, tokens, dtype);
  FX_OK_OR_THROW(fx_kv_store(&c, &r, streamOf(dev)));
  for (const Tensor* t : {&k_cache, &v_cache, &k_scale, &v_scale}) written(*t);
}

std::tuple<Tensor, Tensor> kvRead(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale, const Tensor& slots_,
                                  at::ScalarType dtype) {
  static const char op[] = "functs::kv_read";
  const fx_kv_cache c = cacheOf(op, k_cache, v_cache, k_scale, v_scale);
  const auto dev = k_cache.device();
  const Tensor slots = slotsOf(op, slots_, dev);
  const int32_t tokens = sized(op, slots.numel(), "the number of tokens");
  const int dt = dtypeOf(op, dtype, "dtype");
  c10::DeviceGuard guard(dev);
  Tensor k = at::empty({tokens, c.heads, c.depth}, at::TensorOptions().dtype(dtype).device(dev)), v = at::empty_like(k);
  const fx_kv_rows r = rowsDesc(k, v, slots, tokens, dt);
  FX_OK_OR_THROW(fx_kv_read(&c, &r, streamOf(dev)));
  return {k, v};
}

void attend(const Tensor& q_, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale, const Tensor& block_table,
            const Tensor& lens_, const Tensor& starts_, double scale, int64_t window, int64_t max_new, const Tensor* out_, const Tensor* lse_, Tensor& out,
            Tensor& lse) {
  static const char op[] = "functs::kv_attention";
  const fx_kv_cache c = cacheOf(op, k_cache, v_cache, k_scale, v_scale);
  const auto dev = k_cache.device();
  onGpu(op, q_, "q", dev);
  onGpu(op, block_table, "block_table", dev);
  noGrad(op, q_, "q");
  TORCH_CHECK(q_.dim() == 3 && q_.size(2) == c.depth && q_.size(1) >= 1 && q_.size(1) % c.heads == 0, op, ": q must be [tokens, a multiple of ", c.heads,
              " heads, ", c.depth, "], got ", q_.sizes());
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2, op, ": block_table must be int32 [requests, columns], got ",
              block_table.scalar_type(), " ", block_table.sizes());
  const int64_t B = block_table.size(0);
  TORCH_CHECK(scale >= 0x1p-26 && scale <= 32.0, op, ": scale must lie between 2^-26 and 32, got ", scale);
  TORCH_CHECK(window >= 0 && max_new >= 0, op, ": window and max_new must not be negative, got ", window, " and ", max_new);
  const int dtype = dtypeOf(op, q_.scalar_type(), "q");
  c10::DeviceGuard guard(dev);
  const Tensor lens = ints(op, lens_, "lens", B, dev), starts = ints(op, starts_, "starts", B + 1, dev);
  const Tensor q = q_.stride(2) == 1 ? q_ : q_.contiguous();
  const Tensor table = block_table.size(1) <= 1 || block_table.stride(1) == 1 ? block_table : block_table.contiguous();
  if (out_) {
    onGpu(op, *out_, "out", dev);
    onGpu(op, *lse_, "lse", dev);
    noGrad(op, *out_, "out");
    noGrad(op, *lse_, "lse");
    TORCH_CHECK(out_->scalar_type() == q.scalar_type() && out_->sizes() == q.sizes() && out_->is_contiguous(), op, ": out must be contiguous, of the type and sizes of q");
    TORCH_CHECK(lse_->scalar_type() == at::kFloat && lse_->dim() == 2 && lse_->size(0) == q.size(0) && lse_->size(1) == q.size(1) && lse_->is_contiguous(), op,
                ": lse must be contiguous float32 [tokens, heads]");
    out = *out_;
    lse = *lse_;
  } else {
    out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
    lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  }
  fx_kv_attention_desc d;
  memset(&d, 0, sizeof d);
  d.q = q.data_ptr();
  d.out = out.data_ptr();
  d.lse = lse.data_ptr<float>();
  d.q_token_stride = q.stride(0);
  d.q_head_stride = q.stride(1);
  d.table = table.data_ptr<int32_t>();
  d.table_stride = table.stride(0);
  d.lens = lens.data_ptr<int32_t>();
  d.starts = starts.data_ptr<int32_t>();
  d.tokens = sized(op, q.size(0), "the number of tokens");
  d.requests = sized(op, B, "the number of requests");
  d.columns = sized(op, table.size(1), "the number of columns");
  d.q_heads = sized(op, q.size(1), "the number of heads");
  d.dtype = dtype;
  d.window = (int32_t)std::min<int64_t>(window, INT32_MAX);
  d.max_new = (int32_t)std::min<int64_t>(max_new, INT32_MAX);
  d.clear_rest = out_ ? 0 : 1;
  d.scale = (float)scale;
  // (scratch memory of this call alone, from the allocator of the current stream: calls on other streams and captured
  // graphs have their own)
  const size_t bytes = fx_kv_attention_workspace_bytes(&c, &d);
  TORCH_CHECK(bytes > 0 || d.tokens == 0, "fxhip: ", fx_last_error(), " (", op, ")");
  const Tensor ws = at::empty({(int64_t)std::max<size_t>(bytes, 256)}, at::TensorOptions().dtype(at::kByte).device(dev));
  d.workspace = ws.data_ptr();
  d.workspace_bytes = (size_t)ws.numel();
  FX_OK_OR_THROW(fx_kv_attention(&c, &d, streamOf(dev)));
}

std::tuple<Tensor, Tensor> kvAttention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                                       const Tensor& block_table, const Tensor& lens, const Tensor& starts, double scale, int64_t window, int64_t max_new) {
  Tensor out, lse;
  attend(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, starts, scale, window, max_new, nullptr, nullptr, out, lse);
  return {out, lse};
}
std::tuple<Tensor, Tensor> kvAttentionOut(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                                          const Tensor& block_table, const Tensor& lens, const Tensor& starts, double scale, int64_t window, int64_t max_new,
                                          Tensor out, Tensor lse) {
  Tensor o, l;
  attend(q, k_cache, v_cache, k_scale, v_scale, block_table, lens, starts, scale, window, max_new, &out, &lse, o, l);
  written(out);
  written(lse);
  return {out, lse};
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(functs, m) {
  m.def("kv_plan(Tensor past_lens, Tensor new_lens, Tensor(a!) block_table, Tensor free_pages, int page_size, int max_tokens, "
        "Tensor? free_start=None) -> (Tensor, Tensor, Tensor, Tensor, Tensor)", kvPlan);
  m.def("kv_store(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor slots) -> ()", kvStore);
  m.def("kv_read(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor slots, ScalarType dtype) -> (Tensor, Tensor)", kvRead);
  m.def("kv_attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor block_table, Tensor lens, Tensor starts, "
        "float scale, int window=0, int max_new=0) -> (Tensor, Tensor)", kvAttention);
  m.def("kv_attention.out(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor block_table, Tensor lens, Tensor starts, "
        "float scale, int window=0, int max_new=0, *, Tensor(a!) out, Tensor(b!) lse) -> (Tensor(a!), Tensor(b!))", kvAttentionOut);
}
}  // namespace functs
