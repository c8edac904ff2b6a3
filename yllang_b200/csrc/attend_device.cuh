// What the paged attention kernels share: their parameters, one sequence's
// place in the batch, and the positions that its new tokens see.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "common.cuh"
#include "quant_device.cuh"

namespace ylk {

struct AttnParams {
  const char *q;
  char *o;
  const char *kv[2];
  const float *scale[2];
  const int32_t *kv_indptr, *kv_indices, *last_len, *qo_indptr;
  int64_t q_row_stride, q_head_stride, o_row_stride, o_head_stride;
  int64_t page_stride, slot_stride, head_stride;
  int64_t scale_page_stride, scale_head_stride;
  int64_t indices_cap;
  int64_t num_tokens;
  uint32_t *error_word;
  float *partials;  // decode: unfinished results of the CTAs
  int4 *meta;       // decode: where CTA c's first segment has its parts
  int *items;       // prefill: items taken beyond each CTA's first; the decode kernel before it zeroes it
  int32_t num_pages, batch, heads, group, page_size, window, sinks, max_new;
  int32_t max_rows;  // sequences of at most this many (token, head of a group) rows are the decode kernel's
  FastDiv by_page, by_group;
  float scale_log2;
};

constexpr int64_t kMaxTotal = 1ll << 30;  // tokens of one sequence

// A sequence of the batch.  Its query t is at position first + t.
struct Seq {
  int q0;     // first row of q and o
  int fresh;  // new tokens that have rows in q and o
  int first;  // position of the first new token; below 0 where the sequence has fewer tokens than new ones
  int e0;     // first entry of kv_indices
  int total;  // tokens with the new ones
};

__device__ __forceinline__ Seq load_seq(const AttnParams &p, int i, bool report) {
  Seq s;
  s.q0 = __ldg(p.qo_indptr + i);
  const int64_t fresh = static_cast<int64_t>(__ldg(p.qo_indptr + i + 1)) - s.q0;
  s.e0 = __ldg(p.kv_indptr + i);
  const int64_t pages = static_cast<int64_t>(__ldg(p.kv_indptr + i + 1)) - s.e0;
  const int last = min(max(__ldg(p.last_len + i), 0), p.page_size);
  int64_t total = pages > 0 ? (pages - 1) * p.page_size + last : 0;
  if (total >= kMaxTotal) {
    if (report) raise_deverr(p.error_word, YL_DEVERR_INDPTR_OVERFLOW);
    total = 0;
  }
  s.total = static_cast<int>(total);
  s.first = s.fresh = 0;
  if (fresh <= 0 || s.q0 < 0) return s;
  s.first = static_cast<int>(total - fresh);  // (fresh is below 2^31, as q0 is not negative)
  const bool whole = s.q0 + fresh <= p.num_tokens, fits = p.max_new == 0 || fresh <= p.max_new;
  if (report && !(whole && fits)) raise_deverr(p.error_word, YL_DEVERR_TOKEN_COUNT);
  // rows past the last of q keep those in front of them where they are
  if (fits) s.fresh = static_cast<int>(whole ? fresh : max(p.num_tokens - s.q0, int64_t(0)));
  return s;
}

// The positions that queries [t0, t1) of a sequence see together: [0, head)
// and [low, end), head <= low.
struct Span {
  int head, low, end;
};

__device__ __forceinline__ Span span_of(const AttnParams &p, const Seq &s, int t0, int t1) {
  Span r;
  const int p0 = max(s.first + t0, -1);
  r.end = max(min(s.first + t1, s.total), 0);
  r.low = p.window > 0 ? min(max(0, p0 + 1 - p.window), r.end) : 0;
  r.head = p.window > 0 ? min(p.sinks, r.low) : 0;
  return r;
}

// Whether the query at position pos sees position j.
__device__ __forceinline__ bool sees(const AttnParams &p, int pos, int j) {
  return j <= pos && (p.window == 0 || pos - j < p.window || j < p.sinks);
}

// Neither an infinity nor NaN.
__device__ __forceinline__ bool is_number(float x) { return fabsf(x) < __int_as_float(0x7f800000); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
// 16 bytes, or zeros where !valid.  Written out, so that the load stays in
// flight until its value is used: a conditional expression around __ldg waited
// for it on the spot (8-bit prompt of 8k tokens 690 -> 665 us).
__device__ __forceinline__ uint4 ldg128_if(const void *src, bool valid) {
  uint4 v;
  asm volatile(
      "{\n"
      ".reg .pred q;\n"
      "setp.ne.u32 q, %5, 0;\n"
      "mov.u32 %0, 0;\n"
      "mov.u32 %1, 0;\n"
      "mov.u32 %2, 0;\n"
      "mov.u32 %3, 0;\n"
      "@q ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];\n"
      "}\n"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(src), "r"(static_cast<uint32_t>(valid)));
  return v;
}
// Arrive on `bar` (no count added) once this thread's earlier cp.async have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Lets a kernel have `bytes` of dynamic shared memory on the current device
// (asked for once per kernel and device); a yl_status.
int allow_smem(const void *fn, int bytes);

// The decode kernel: workspace bytes, and its launch for sequences of at most
// p.max_rows query rows per KV head, none of which has more than most_rows.
int64_t decode_workspace(const yl_paged_attention_args *a, int64_t most_rows);
int launch_decode(AttnParams &p, const yl_paged_attention_args *a, int64_t most_rows, cudaStream_t stream);
// The prefill kernel, for sequences of more than p.max_rows rows.
int launch_prefill(AttnParams &p, const yl_paged_attention_args *a, cudaStream_t stream);

}  // namespace ylk
