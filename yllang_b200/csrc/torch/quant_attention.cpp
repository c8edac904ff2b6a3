// Front end of the 8-bit pool and of the paged attention: shape checks and
// strides on top of yl_kv_quant_store, yl_kv_quant_load and yl_paged_attention.
#include <climits>

#include "frontend.h"
#include "yl_kvpath.h"
#include "yllang_kvpath.h"

namespace yllang {
namespace {

// RuntimeCheck whose message is made only when it is thrown: these calls run
// once per layer of a step.
#define YL_REQUIRE(cond, what, message) \
  if (!(cond)) throw PanicError(std::string(what) + ": " + (message))

std::string Shape(const torch::Tensor &t) {
  std::ostringstream os;
  os << t.sizes();
  return os.str();
}

int DtypeOf(const torch::Tensor &t, const char *what, const char *name) {
  const auto st = t.scalar_type();
  YL_REQUIRE(st == torch::kBFloat16 || st == torch::kHalf, what, std::string(name) + " must be bf16 or fp16");
  return st == torch::kBFloat16 ? YL_DTYPE_BF16 : YL_DTYPE_F16;
}

yl_quant_pool PoolArgs(const QuantKVPool &pool, const char *what) {
  const auto &k = pool.k, &v = pool.v, &ks = pool.k_scale, &vs = pool.v_scale;
  const int64_t d = k.dim();
  YL_REQUIRE(d == 4 || d == 5, what, "pool.k must be [P, page_size, H, D] or [L, P, page_size, H, D], got " + Shape(k));
  YL_REQUIRE(k.is_cuda(), what, "the pool must be CUDA tensors");
  YL_REQUIRE(k.scalar_type() == torch::kFloat8_e4m3fn && v.scalar_type() == torch::kFloat8_e4m3fn, what,
             "pool.k and pool.v must be float8_e4m3fn");
  YL_REQUIRE(v.sizes() == k.sizes() && v.strides() == k.strides(), what, "pool.k and pool.v must share shape and strides");
  YL_REQUIRE(k.stride(-1) == 1, what, "head rows must be contiguous");
  YL_REQUIRE(ks.scalar_type() == torch::kFloat32 && vs.scalar_type() == torch::kFloat32, what, "scales must be fp32");
  const bool layers = d == 5;
  YL_REQUIRE(ks.dim() == d - 2 && ks.size(-1) == k.size(-2) && ks.size(-2) == k.size(-4) &&
                 (!layers || ks.size(0) == k.size(0)) && vs.sizes() == ks.sizes() && vs.strides() == ks.strides(),
             what, "scales must be [P, H], with the pool's layers in front, and share strides");
  YL_REQUIRE(v.device() == k.device() && ks.device() == k.device() && vs.device() == k.device(), what,
             "the pool's tensors must be on one device");
  yl_quant_pool a{};
  a.k_codes = k.data_ptr();
  a.v_codes = v.data_ptr();
  a.k_scale = ks.data_ptr<float>();
  a.v_scale = vs.data_ptr<float>();
  a.page_stride = k.stride(-4);
  a.slot_stride = k.stride(-3);
  a.head_stride = k.stride(-2);
  a.scale_page_stride = ks.stride(-2);
  a.scale_head_stride = ks.stride(-1);
  a.num_layers = 1;
  if (layers) {
    YL_REQUIRE(k.size(0) <= INT_MAX, what, "too many layers");
    a.num_layers = static_cast<int32_t>(k.size(0));
    a.layer_stride = k.stride(0);
    a.scale_layer_stride = ks.stride(0);
  }
  YL_REQUIRE(k.size(-3) <= INT_MAX && k.size(-2) <= INT_MAX, what, "page_size or heads out of range");
  a.num_pages = k.size(-4);
  a.page_size = static_cast<int32_t>(k.size(-3));
  a.num_heads = static_cast<int32_t>(k.size(-2));
  a.head_dim = static_cast<int32_t>(k.size(-1));
  return a;
}

// K/V rows beside a pool: [N, H*D] or [N, H, D], with the pool's layers in front.
struct Rows {
  int64_t tokens, row_stride, layer_stride;  // strides in bytes
};
Rows RowsOf(const torch::Tensor &t, const QuantKVPool &pool, const char *what, const char *name) {
  const int64_t lead = pool.k.dim() - 4, h = pool.k.size(-2), d = pool.k.size(-1);
  const int64_t row = t.dim() - lead - 1;  // dimensions of a row
  const bool ok = (row == 1 && t.size(-1) == h * d) || (row == 2 && t.size(-2) == h && t.size(-1) == d);
  YL_REQUIRE(ok && (lead == 0 || t.size(0) == pool.k.size(0)), what,
             std::string(name) + " must be [N, H*D] or [N, H, D] rows, with the pool's layers in front, got " + Shape(t));
  YL_REQUIRE(t.stride(-1) == 1 && (row == 1 || h == 1 || t.stride(-2) == d), what,
             std::string(name) + " rows must be contiguous");
  const int64_t n = t.size(lead);
  // a single row's stride means nothing: give the kernel a valid one
  return {n, 2 * (n > 1 ? t.stride(lead) : h * d), lead ? 2 * t.stride(0) : 0};
}

int64_t CheckIndex(const BatchIndex &index, const torch::Device &device, const char *what) {
  for (const auto *t : {&index.kv_indptr, &index.kv_indices, &index.kv_last_page_len, &index.qo_indptr})
    YL_REQUIRE(t->scalar_type() == torch::kInt32 && t->dim() == 1 && t->is_contiguous() && t->device() == device, what,
               "index: kv_indptr, kv_indices, kv_last_page_len and qo_indptr must be contiguous int32 on the call's device");
  const int64_t b = index.kv_indptr.size(0) - 1;
  YL_REQUIRE(b >= 0 && b <= INT_MAX && index.qo_indptr.size(0) == b + 1 && index.kv_last_page_len.size(0) >= b, what,
             "index needs kv_indptr and qo_indptr [B + 1] and kv_last_page_len [B]");
  return b;
}

}  // namespace

QuantKVPool MakeQuantKVPool(int64_t num_pages, int64_t page_size, int64_t num_kv_heads, int64_t head_dim,
                            int64_t num_layers, torch::Device device) {
  RuntimeCheck(num_pages > 0 && page_size > 0 && num_kv_heads > 0 && head_dim > 0 && num_layers >= 0,
               "MakeQuantKVPool: sizes must be positive");
  std::vector<int64_t> shape{num_pages, num_kv_heads, page_size, head_dim}, scales{num_pages, num_kv_heads};
  if (num_layers > 0) {
    shape.insert(shape.begin(), num_layers);
    scales.insert(scales.begin(), num_layers);
  }
  const auto codes = [&] {
    return torch::zeros(shape, torch::dtype(torch::kUInt8).device(device)).view(torch::kFloat8_e4m3fn).transpose(-3, -2);
  };
  const auto ones = [&] { return torch::ones(scales, torch::dtype(torch::kFloat32).device(device)); };
  return {codes(), codes(), ones(), ones()};
}

void StoreKVCacheQuant(const torch::Tensor &k, const torch::Tensor &v, const QuantKVPool &pool, const BatchIndex &index,
                       const std::optional<torch::Tensor> &error_word) {
  const char *what = "StoreKVCacheQuant";
  const Range range("yllang::StoreKVCacheQuant");
  yl_quant_store_args a{};
  a.pool = PoolArgs(pool, what);
  a.dtype = DtypeOf(k, what, "k");
  YL_REQUIRE(v.scalar_type() == k.scalar_type(), what, "k and v must share their dtype");
  const auto device = pool.k.device();
  YL_REQUIRE(k.device() == device && v.device() == device, what, "k and v must be on the pool's device");
  const Rows kr = RowsOf(k, pool, what, "k"), vr = RowsOf(v, pool, what, "v");
  YL_REQUIRE(kr.tokens == vr.tokens, what, "k and v must have the same rows");
  const int64_t b = CheckIndex(index, device, what);
  const DeviceErrorScope errors(device, ErrorWordOf(error_word, device, what), what);
  if (kr.tokens == 0 || b == 0) return;
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.kv_indptr = index.kv_indptr.data_ptr<int32_t>();
  a.kv_indices = index.kv_indices.data_ptr<int32_t>();
  a.kv_last_page_len = index.kv_last_page_len.data_ptr<int32_t>();
  a.qo_indptr = index.qo_indptr.data_ptr<int32_t>();
  a.kv_indices_capacity = index.kv_indices.size(0);
  a.num_tokens = kr.tokens;
  a.k_row_stride = kr.row_stride;
  a.v_row_stride = vr.row_stride;
  a.k_layer_stride = kr.layer_stride;
  a.v_layer_stride = vr.layer_stride;
  a.batch_size = static_cast<int32_t>(b);
  a.error_word = errors.word();
  const c10::cuda::CUDAGuard guard(device);
  CheckStatus(yl_kv_quant_store(&a, CurrentStream(k)), "yl_kv_quant_store");
  errors.Check();
}

std::pair<torch::Tensor, torch::Tensor> LoadKVCacheQuant(const QuantKVPool &pool, const torch::Tensor &slots,
                                                         torch::Dtype dtype,
                                                         const std::optional<std::pair<torch::Tensor, torch::Tensor>> &out,
                                                         const std::optional<torch::Tensor> &error_word) {
  const char *what = "LoadKVCacheQuant";
  const Range range("yllang::LoadKVCacheQuant");
  yl_quant_load_args a{};
  a.pool = PoolArgs(pool, what);
  const auto device = pool.k.device();
  YL_REQUIRE(slots.dim() == 1 && (slots.scalar_type() == torch::kInt32 || slots.scalar_type() == torch::kInt64) &&
                 slots.device() == device && (slots.size(0) <= 1 || slots.stride(0) == 1),
             what, "slots must be contiguous int32 or int64 [N] on the pool's device");
  const int64_t n = slots.size(0);
  std::pair<torch::Tensor, torch::Tensor> kv;
  if (out) {
    kv = *out;
  } else {
    YL_REQUIRE(dtype == torch::kBFloat16 || dtype == torch::kHalf, what, "dtype must be bf16 or fp16");
    std::vector<int64_t> shape{n, a.pool.num_heads, a.pool.head_dim};
    if (pool.k.dim() == 5) shape.insert(shape.begin(), a.pool.num_layers);
    const auto options = torch::dtype(dtype).device(device);
    kv = {torch::empty(shape, options), torch::empty(shape, options)};
  }
  a.dtype = DtypeOf(kv.first, what, "out");
  YL_REQUIRE(kv.second.scalar_type() == kv.first.scalar_type() && kv.first.device() == device && kv.second.device() == device,
             what, "out must be two bf16 or two fp16 tensors on the pool's device");
  const Rows kr = RowsOf(kv.first, pool, what, "out k"), vr = RowsOf(kv.second, pool, what, "out v");
  YL_REQUIRE(kr.tokens == n && vr.tokens == n, what, "out must have a row for each slot");
  const DeviceErrorScope errors(device, ErrorWordOf(error_word, device, what), what);
  if (n == 0) return kv;
  a.k_out = kv.first.data_ptr();
  a.v_out = kv.second.data_ptr();
  a.slots = slots.data_ptr();
  a.num_tokens = n;
  a.k_row_stride = kr.row_stride;
  a.v_row_stride = vr.row_stride;
  a.k_layer_stride = kr.layer_stride;
  a.v_layer_stride = vr.layer_stride;
  a.slot_is_int64 = slots.scalar_type() == torch::kInt64 ? 1 : 0;
  a.error_word = errors.word();
  const c10::cuda::CUDAGuard guard(device);
  CheckStatus(yl_kv_quant_load(&a, CurrentStream(pool.k)), "yl_kv_quant_load");
  errors.Check();
  return kv;
}

namespace {
yl_paged_attention_args AttentionArgs(const torch::Tensor &q, const torch::Tensor &k, const torch::Tensor &v,
                                      const BatchIndex &index, const PagedAttentionOptions &o, const char *what) {
  yl_paged_attention_args a{};
  YL_REQUIRE(q.dim() == 3 && q.stride(2) == 1, what, "q must be [N, Hq, head_dim] with contiguous heads");
  YL_REQUIRE(q.is_cuda(), what, "q must be a CUDA tensor");
  a.dtype = DtypeOf(q, what, "q");
  const auto device = q.device();
  YL_REQUIRE(k.dim() == 4 && k.stride(3) == 1, what, "k_pages must be [P, page_size, H, D] with contiguous head rows");
  YL_REQUIRE(v.sizes() == k.sizes() && v.strides() == k.strides() && v.scalar_type() == k.scalar_type(), what,
             "k_pages and v_pages must share shape, strides and dtype");
  YL_REQUIRE(k.device() == device && v.device() == device, what, "the pool must be on q's device");
  const int64_t pages = k.size(0), page_size = k.size(1), heads = k.size(2), d = q.size(2), qheads = q.size(1);
  YL_REQUIRE(k.size(3) == d, what, "head_dim of the pool differs from q's");
  YL_REQUIRE(heads > 0 && qheads > 0 && qheads % heads == 0 && qheads <= INT_MAX, what,
             "query heads must be a multiple of the KV heads");
  YL_REQUIRE(page_size <= INT_MAX, what, "page_size out of range");
  const int64_t item = k.element_size();
  if (k.scalar_type() == torch::kFloat8_e4m3fn) {
    YL_REQUIRE(o.k_scale && o.v_scale, what, "an 8-bit pool needs k_scale and v_scale");
    for (const auto *s : {&*o.k_scale, &*o.v_scale})
      YL_REQUIRE(s->scalar_type() == torch::kFloat32 && s->dim() == 2 && s->size(0) == pages && s->size(1) == heads &&
                     s->device() == device,
                 what, "k_scale and v_scale must be fp32 [P, H] on q's device");
    YL_REQUIRE(o.k_scale->strides() == o.v_scale->strides(), what, "k_scale and v_scale must share strides");
    a.k_scale = o.k_scale->data_ptr<float>();
    a.v_scale = o.v_scale->data_ptr<float>();
    a.scale_page_stride = o.k_scale->stride(0);
    a.scale_head_stride = o.k_scale->stride(1);
    a.kv_dtype = YL_KV_E4M3;
  } else {
    YL_REQUIRE(k.scalar_type() == q.scalar_type(), what, "the pool must be float8_e4m3fn or of q's dtype");
    YL_REQUIRE(!o.k_scale && !o.v_scale, what, "scales are for 8-bit pools");
    a.kv_dtype = YL_KV_SAME;
  }
  const int64_t b = CheckIndex(index, device, what);
  YL_REQUIRE(o.window >= 0 && o.window <= INT_MAX && o.sinks >= 0 && o.sinks <= INT_MAX && o.max_new_len >= 0 &&
                 o.max_new_len <= INT_MAX,
             what, "window, sinks and max_new_len must be in [0, 2^31)");
  a.q = q.data_ptr();
  a.k_cache = k.data_ptr();
  a.v_cache = v.data_ptr();
  a.kv_indptr = index.kv_indptr.data_ptr<int32_t>();
  a.kv_indices = index.kv_indices.data_ptr<int32_t>();
  a.kv_last_page_len = index.kv_last_page_len.data_ptr<int32_t>();
  a.qo_indptr = index.qo_indptr.data_ptr<int32_t>();
  a.q_row_stride = 2 * (q.size(0) > 1 ? q.stride(0) : qheads * d);
  a.q_head_stride = 2 * (qheads > 1 ? q.stride(1) : d);
  // the stride of a dimension of one means nothing
  a.page_stride = item * (pages > 1 ? k.stride(0) : page_size * heads * d);
  a.slot_stride = item * (page_size > 1 ? k.stride(1) : heads * d);
  a.head_stride = item * (heads > 1 ? k.stride(2) : d);
  a.kv_indices_capacity = index.kv_indices.size(0);
  a.num_pages = pages;
  a.num_tokens = q.size(0);
  a.batch_size = static_cast<int32_t>(b);
  a.num_q_heads = static_cast<int32_t>(qheads);
  a.num_kv_heads = static_cast<int32_t>(heads);
  a.head_dim = static_cast<int32_t>(d);
  a.page_size = static_cast<int32_t>(page_size);
  a.window = static_cast<int32_t>(o.window);
  a.sinks = static_cast<int32_t>(o.sinks);
  a.max_new_len = static_cast<int32_t>(o.max_new_len);
  a.sm_scale = static_cast<float>(o.sm_scale ? *o.sm_scale : 1.0 / std::sqrt(static_cast<double>(d)));
  return a;
}

int64_t WorkspaceOf(const yl_paged_attention_args &a) {
  const int64_t need = yl_paged_attention_workspace(&a);
  if (need < 0) CheckStatus(static_cast<int>(need), "yl_paged_attention");
  return need;
}
}  // namespace

int64_t PagedAttentionWorkspace(const torch::Tensor &q, const torch::Tensor &k_pages, const torch::Tensor &v_pages,
                                const BatchIndex &index, const PagedAttentionOptions &options) {
  const auto a = AttentionArgs(q, k_pages, v_pages, index, options, "PagedAttentionWorkspace");
  const c10::cuda::CUDAGuard guard(q.device());
  return WorkspaceOf(a);
}

torch::Tensor PagedAttention(const torch::Tensor &q, const torch::Tensor &k_pages, const torch::Tensor &v_pages,
                             const BatchIndex &index, const PagedAttentionOptions &options) {
  const char *what = "PagedAttention";
  const Range range("yllang::PagedAttention");
  auto a = AttentionArgs(q, k_pages, v_pages, index, options, what);
  const auto device = q.device();
  const c10::cuda::CUDAGuard guard(device);
  torch::Tensor out = options.out ? *options.out : torch::empty(q.sizes(), q.options());
  YL_REQUIRE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == device && out.stride(2) == 1,
             what, "out must be like q, with contiguous heads");
  const DeviceErrorScope errors(device, ErrorWordOf(options.error_word, device, what), what);
  if (a.num_tokens == 0 || a.batch_size == 0) return out;
  a.o = out.data_ptr();
  a.o_row_stride = 2 * (a.num_tokens > 1 ? out.stride(0) : a.num_q_heads * static_cast<int64_t>(a.head_dim));
  a.o_head_stride = 2 * (a.num_q_heads > 1 ? out.stride(1) : a.head_dim);
  const int64_t need = WorkspaceOf(a);
  torch::Tensor workspace;
  if (options.workspace) {
    workspace = *options.workspace;
    YL_REQUIRE(workspace.scalar_type() == torch::kUInt8 && workspace.is_contiguous() && workspace.device() == device &&
                   workspace.numel() >= need,
               what, "workspace must be " + std::to_string(need) + " contiguous bytes on q's device");
  } else {
    workspace = torch::empty({need}, torch::dtype(torch::kUInt8).device(device));
  }
  a.workspace = workspace.data_ptr();
  a.workspace_bytes = workspace.numel();
  a.error_word = errors.word();
  CheckStatus(yl_paged_attention(&a, CurrentStream(q)), "yl_paged_attention");
  errors.Check();
  return out;
}

}  // namespace yllang
