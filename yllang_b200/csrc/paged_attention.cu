// yl_paged_attention: argument checks, and which kernel takes which sequence of
// the batch (attend_decode.cu, attend_prefill.cu).
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <map>
#include <mutex>

#include "attend_device.cuh"

namespace ylk {
namespace {

// Query rows per KV head (new tokens times heads of the group) up to which a
// sequence is the decode kernel's.  It reads the keys once for each 16 rows, in
// parts over all SMs; the prefill kernel once for 256, by one SM.  32 sequences
// of up to 8k tokens, 8-bit, 8 KV heads of 128: 32 rows 152 us against 324, 64
// rows 286 against 332, 128 rows 556 against 331.  The rule looks at a sequence's
// rows only: one sequence alone, whose items are fewer than the SMs, loses by it
// (at 128 rows 119 us, 35 in the decode kernel).
constexpr int kDecodeRows = 64;

// Most query rows per KV head that a sequence of the call can have.
int64_t most_rows(const yl_paged_attention_args *a) {
  const int64_t fresh = a->max_new_len > 0 ? std::min<int64_t>(a->max_new_len, a->num_tokens) : a->num_tokens;
  return fresh * (a->num_q_heads / a->num_kv_heads);
}

int check_attention(const yl_paged_attention_args *a, bool pointers) {
  if (a == nullptr) return fail(YL_ERR_NULL_ARG, "yl_paged_attention: args is NULL");
  if (a->batch_size < 0) return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: batch_size=%lld < 0", a->batch_size);
  if (a->num_tokens < 0) return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: num_tokens=%lld < 0", a->num_tokens);
  if (a->num_tokens >= (1ll << 31))
    return fail(YL_ERR_UNSUPPORTED, "yl_paged_attention: num_tokens=%lld must be below 2^31", a->num_tokens);
  if (a->dtype != YL_DTYPE_BF16 && a->dtype != YL_DTYPE_F16)
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: dtype=%lld unknown", a->dtype);
  if (a->kv_dtype != YL_KV_SAME && a->kv_dtype != YL_KV_E4M3)
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: kv_dtype=%lld unknown", a->kv_dtype);
  if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256)
    return fail(YL_ERR_UNSUPPORTED, "yl_paged_attention: head_dim=%lld must be 64, 128 or 256", a->head_dim);
  if (a->num_kv_heads < 1 || a->num_q_heads < 1 || a->num_q_heads % a->num_kv_heads != 0)
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: num_q_heads=%lld must be a multiple of num_kv_heads=%lld",
                a->num_q_heads, a->num_kv_heads);
  if (a->num_tokens * (a->num_q_heads / a->num_kv_heads) >= (1ll << 31))
    return fail(YL_ERR_UNSUPPORTED, "yl_paged_attention: num_tokens=%lld times the group passes 2^31", a->num_tokens);
  if (a->num_kv_heads > 32767)
    return fail(YL_ERR_UNSUPPORTED, "yl_paged_attention: num_kv_heads=%lld exceeds 32767", a->num_kv_heads);
  if (a->page_size < 1) return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: page_size=%lld < 1", a->page_size);
  if (a->window < 0 || a->sinks < 0 || a->max_new_len < 0)
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: window, sinks and max_new_len must not be negative");
  if (!(a->sm_scale > 0.f) || !(a->sm_scale <= 3.0e38f))
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: sm_scale must be positive and finite");
  if (a->kv_indices_capacity < 0)
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: kv_indices_capacity=%lld < 0", a->kv_indices_capacity);
  if (a->num_pages < 1 || a->num_pages >= (1ll << 31))
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: num_pages=%lld must be in [1, 2^31)", a->num_pages);
  if (!pointers || a->batch_size == 0 || a->num_tokens == 0) return YL_OK;
  const int64_t item = a->kv_dtype == YL_KV_E4M3 ? 1 : 2;
  if (!a->q || !a->o || !a->k_cache || !a->v_cache || !a->kv_indptr || !a->kv_last_page_len || !a->qo_indptr ||
      (!a->kv_indices && a->kv_indices_capacity > 0))
    return fail(YL_ERR_NULL_ARG, "yl_paged_attention: q, o, the pool and the page arrays must be non-NULL");
  if (a->kv_dtype == YL_KV_E4M3 && (!a->k_scale || !a->v_scale))
    return fail(YL_ERR_NULL_ARG, "yl_paged_attention: an 8-bit pool needs k_scale and v_scale");
  if (a->q_head_stride < a->head_dim * 2 || a->o_head_stride < a->head_dim * 2 || a->q_row_stride < a->head_dim * 2 ||
      a->o_row_stride < a->head_dim * 2 || a->slot_stride < a->head_dim * item ||
      a->head_stride < a->head_dim * item || a->page_stride < a->head_dim * item)
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: strides must be at least one head row of %lld elements",
                a->head_dim);
  if (a->kv_dtype == YL_KV_E4M3 && (a->scale_page_stride < 1 || a->scale_head_stride < 1))
    return fail(YL_ERR_BAD_SIZE, "yl_paged_attention: scale strides must be positive");
  const uintptr_t bits =
      reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->o) | reinterpret_cast<uintptr_t>(a->k_cache) |
      reinterpret_cast<uintptr_t>(a->v_cache) |
      static_cast<uintptr_t>(a->q_row_stride | a->q_head_stride | a->o_row_stride | a->o_head_stride |
                             a->page_stride | a->slot_stride | a->head_stride);
  if (bits & 15u)
    return fail(YL_ERR_ALIGNMENT, "yl_paged_attention: pointers and strides of q, o and the pool must be multiples of "
                                  "16 bytes");
  const uintptr_t words =
      reinterpret_cast<uintptr_t>(a->kv_indptr) | reinterpret_cast<uintptr_t>(a->kv_indices) |
      reinterpret_cast<uintptr_t>(a->kv_last_page_len) | reinterpret_cast<uintptr_t>(a->qo_indptr) |
      reinterpret_cast<uintptr_t>(a->error_word) |
      (a->kv_dtype == YL_KV_E4M3 ? reinterpret_cast<uintptr_t>(a->k_scale) | reinterpret_cast<uintptr_t>(a->v_scale) : 0);
  if (words & 3u)
    return fail(YL_ERR_ALIGNMENT, "yl_paged_attention: page arrays, scales and error_word must be 4-byte aligned");
  return YL_OK;
}

}  // namespace

int allow_smem(const void *fn, int bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, const void *>, int> done;
  std::lock_guard<std::mutex> lock(mu);
  int &have = done[std::make_pair(current_device(), fn)];
  if (have >= bytes) return YL_OK;
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_error(std::string("yl_paged_attention: shared memory: ") + cudaGetErrorString(e));
    return YL_ERR_CUDA;
  }
  have = bytes;
  return YL_OK;
}

}  // namespace ylk

extern "C" int64_t yl_paged_attention_workspace(const yl_paged_attention_args *a) {
  using namespace ylk;
  clear_last_error();
  const int rc = check_attention(a, false);
  return rc != YL_OK ? rc : decode_workspace(a, most_rows(a));
}

extern "C" int yl_paged_attention(const yl_paged_attention_args *a, cudaStream_t stream) {
  using namespace ylk;
  clear_last_error();
  int rc = check_attention(a, true);
  if (rc != YL_OK) return rc;
  if (a->batch_size == 0 || a->num_tokens == 0) return YL_OK;
  const int64_t most = most_rows(a);
  if (a->workspace == nullptr || a->workspace_bytes < decode_workspace(a, most))
    return fail(a->workspace ? YL_ERR_BAD_SIZE : YL_ERR_NULL_ARG,
                "yl_paged_attention: workspace must hold %lld bytes", decode_workspace(a, most));
  if (reinterpret_cast<uintptr_t>(a->workspace) & 15u)
    return fail(YL_ERR_ALIGNMENT, "yl_paged_attention: workspace must be 16-byte aligned");
  AttnParams p;
  p.q = static_cast<const char *>(a->q);
  p.o = static_cast<char *>(a->o);
  p.kv[0] = static_cast<const char *>(a->k_cache);
  p.kv[1] = static_cast<const char *>(a->v_cache);
  p.scale[0] = a->k_scale;
  p.scale[1] = a->v_scale;
  p.kv_indptr = a->kv_indptr;
  p.kv_indices = a->kv_indices;
  p.last_len = a->kv_last_page_len;
  p.qo_indptr = a->qo_indptr;
  p.q_row_stride = a->q_row_stride;
  p.q_head_stride = a->q_head_stride;
  p.o_row_stride = a->o_row_stride;
  p.o_head_stride = a->o_head_stride;
  p.page_stride = a->page_stride;
  p.slot_stride = a->slot_stride;
  p.head_stride = a->head_stride;
  p.scale_page_stride = a->scale_page_stride;
  p.scale_head_stride = a->scale_head_stride;
  p.indices_cap = a->kv_indices_capacity;
  p.num_tokens = a->num_tokens;
  p.error_word = a->error_word;
  p.num_pages = static_cast<int32_t>(a->num_pages);
  p.batch = a->batch_size;
  p.heads = a->num_kv_heads;
  p.group = a->num_q_heads / a->num_kv_heads;
  p.page_size = a->page_size;
  p.window = std::min(a->window, 1 << 30);  // (no sequence is longer; positions minus it stay in 32 bits)
  p.sinks = a->sinks;
  p.max_new = a->max_new_len;
  p.by_page = FastDiv(static_cast<uint32_t>(a->page_size));
  p.by_group = FastDiv(static_cast<uint32_t>(p.group));
  p.scale_log2 = a->sm_scale * 1.44269504088896f;
  p.max_rows = kDecodeRows;
  rc = launch_decode(p, a, most, stream);
  if (rc != YL_OK || most <= kDecodeRows) return rc;
  return launch_prefill(p, a, stream);
}
