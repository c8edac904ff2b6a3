// The 8-bit pool's store and load, for sm_100a: K/V rows quantised to e4m3 as
// they are written, one power-of-two scale for each (page, head), and read
// back by slot.
//
// Store.  Work item = (page that gets new tokens, head, plane), plane = 2 *
// layer + {K, V}: nothing else of the call writes that block, so its scale
// needs no atomics and the result does not depend on any order.  A lane group
// of head_dim / 8 lanes owns an item: each lane holds 8 elements of every new
// token's row (16-byte loads), the group's running maximum is taken on the bit
// patterns of |x| (ordered like the values, infinities and NaN on top), then
// the rows are scaled and written from the registers.  The neighbouring groups
// of a warp take neighbouring heads, so the warp reads whole 512-byte runs of
// the token-major input.  A warp finds its page once (a 32-way search over the
// batch) and walks its planes.
//
// Algorithmic bytes per element: 2 read + 1 written for the store, 1 read + 2
// written for the load, so HBM bounds both.  Measured, bf16 rows of 8 heads of
// 128: a prompt step of 64 sequences, 32 layers, 269 us, 6.75 TB/s, as fast as a
// plain copy; a decode step of 256 sequences, 32 layers, 22.3 us, 2.3 TB/s (two
// rounds of eight planes a warp, and 213 instructions per 512 bytes of rows, 60 %
// of the issue slots); pages of one token 937 us for the same prompts; 131,072
// tokens of one layer read back in 154 us, 5.2 TB/s, where two bytes in three are
// writes and a fill of the same memory reaches 3.9 TB/s.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "common.cuh"
#include "quant_device.cuh"

namespace ylk {
namespace {

struct QuantPool {
  uint8_t *codes[2];
  float *scale[2];
  int64_t layer_stride, page_stride, slot_stride, head_stride;
  int64_t scale_layer_stride, scale_page_stride, scale_head_stride;
  int32_t num_pages, page_size, num_heads;
};

struct QuantStoreParams {
  QuantPool pool;
  const char *x[2];
  int64_t row_stride[2], layer_stride[2];
  const int32_t *kv_indptr, *kv_indices, *last_len, *qo_indptr;
  int64_t indices_cap, num_tokens;
  uint32_t *error_word;
  int32_t batch, planes;
  uint32_t cands, chunks, runs, planes_per_run;
};

constexpr int kStoreThreads = 128;

// The pages that a batch touches, numbered without a scan.  By token: number n
// is the page of row n if n is the first new token in it.  By page: sequence
// i's pages get the numbers from qo_indptr[i] / page_size + 2 i on; it touches
// at most (new - 1) / page_size + 2 pages, which that leaves room for.  The
// host takes whichever numbering is shorter.
struct Touched {
  int64_t page;
  int64_t row0;  // first row of k and v
  int held;      // tokens the page had
  int count;     // new tokens of the page; 0: nothing to do
};

// Rows that k and v lack may be nobody's number: the last number, found in
// sequence i, which ends at row q1, looks for them.  (A call of its own: the two
// compares inline cost a decode step of 256 sequences 0.2 us, a warp beyond the
// units 0.3 of 22.4.)
__device__ __noinline__ void look_behind(const QuantStoreParams &p, int64_t q1, int i) {
  if (q1 > p.num_tokens || (i + 1 < p.batch && __ldg(p.qo_indptr + p.batch) > p.num_tokens))
    raise_deverr(p.error_word, YL_DEVERR_TOKEN_COUNT);
}

template <bool BY_TOKEN>
__device__ __forceinline__ Touched find_page(const QuantStoreParams &p, uint32_t cand, int lane, bool report) {
  Touched r;
  r.count = 0;
  r.page = r.row0 = 0;
  r.held = 0;
  const int ps = p.pool.page_size;
  int i = 0;
  int64_t q0, q1, e0, e1;
  int last;
  auto load = [&]() {
    q0 = __ldg(p.qo_indptr + i);
    q1 = __ldg(p.qo_indptr + i + 1);
    e0 = __ldg(p.kv_indptr + i);
    e1 = __ldg(p.kv_indptr + i + 1);
    last = __ldg(p.last_len + i);
  };
  if (BY_TOKEN) {
    // in a decode batch row n is sequence n's, which saves the search's loads
    i = static_cast<int>(min(cand, static_cast<uint32_t>(p.batch - 1)));
    load();
  }
  if (!BY_TOKEN || q0 > cand || q1 <= cand) {
    i = warp_find(p.batch, cand, lane, [&](int s) -> int64_t {
      const int64_t q = __ldg(p.qo_indptr + s);
      return BY_TOKEN ? q : q / ps + 2ll * s;
    });
    load();
  }
  if (cand + 1 == p.cands) look_behind(p, q1, i);
  const int64_t fresh = q1 - q0, pages = e1 - e0;
  if (fresh <= 0 || q0 < 0) return r;
  last = min(max(last, 0), ps);
  const int64_t total = pages > 0 ? (pages - 1) * ps + last : 0;
  const int64_t prior = total - fresh;
  int64_t ord;
  if (BY_TOKEN) {
    const int64_t t = static_cast<int64_t>(cand) - q0;
    const int64_t pos = prior + t;
    if (t < 0 || t >= fresh) return r;  // a row in front of the first sequence, or behind the last
    if (prior < 0 && t == 0 && report) raise_deverr(p.error_word, YL_DEVERR_ROW_OVERFLOW);
    if (pos < 0 || (t > 0 && pos % ps != 0)) return r;
    ord = pos / ps;
  } else {
    const int64_t j = static_cast<int64_t>(cand) - (q0 / ps + 2ll * i);
    if (prior < 0 && j == 0 && report) raise_deverr(p.error_word, YL_DEVERR_ROW_OVERFLOW);
    ord = max(prior, int64_t(0)) / ps + j;
  }
  const int64_t a = max(max(prior, int64_t(0)), ord * ps), b = min(total, (ord + 1) * ps);
  if (a >= b) return r;
  int64_t n = b - a;
  r.row0 = q0 + (a - prior);
  if (r.row0 + n > p.num_tokens) {
    if (report) raise_deverr(p.error_word, YL_DEVERR_TOKEN_COUNT);
    n = max(p.num_tokens - r.row0, int64_t(0));
  }
  const int64_t e = e0 + ord;
  if (e < 0 || e >= p.indices_cap) {
    if (report) raise_deverr(p.error_word, YL_DEVERR_INDICES_CAP);
    return r;
  }
  const int64_t page = __ldg(p.kv_indices + e);
  if (page < 0 || page >= p.pool.num_pages) {
    if (report) raise_deverr(p.error_word, YL_DEVERR_PAGE_RANGE);
    return r;
  }
  r.page = page;
  r.held = static_cast<int>(a - ord * ps);
  r.count = static_cast<int>(n);
  return r;
}

// Running maximum of |x| as bit patterns of 16-bit pairs.
__device__ __forceinline__ uint32_t abs_max8(uint32_t m, const uint4 &w) {
  m = __vmaxu2(m, w.x & 0x7fff7fffu);
  m = __vmaxu2(m, w.y & 0x7fff7fffu);
  m = __vmaxu2(m, w.z & 0x7fff7fffu);
  return __vmaxu2(m, w.w & 0x7fff7fffu);
}

template <typename T>
__device__ __forceinline__ float finite_abs_max8(float m, const uint4 &w) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::unpack(v[i]);
    if (fabsf(f.x) <= T::kMax) m = fmaxf(m, fabsf(f.x));
    if (fabsf(f.y) <= T::kMax) m = fmaxf(m, fabsf(f.y));
  }
  return m;
}

template <typename T>
__device__ __forceinline__ uint2 quantise8(const uint4 &w, float inv) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = T::unpack(v[i]);
    c[i] = float2_to_e4m3x2(f.x * inv, f.y * inv);
  }
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

// Held tokens take the page's new scale (each code times old / new, rounded).
__device__ __forceinline__ void requantise(uint8_t *codes, int64_t slot_stride, int first, int held, int step, float ratio) {
  for (int t = first; t < held; t += step) {
    uint2 *at = reinterpret_cast<uint2 *>(codes + t * slot_stride);
    const uint2 w = *at;
    const uint32_t v[2] = {w.x, w.y};
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 lo = half2_bits_to_float2(e4m3x2_to_half2(static_cast<uint16_t>(v[i] & 0xffffu)));
      const float2 hi = half2_bits_to_float2(e4m3x2_to_half2(static_cast<uint16_t>(v[i] >> 16)));
      c[i] = float2_to_e4m3x2(lo.x * ratio, lo.y * ratio) |
             static_cast<uint32_t>(float2_to_e4m3x2(hi.x * ratio, hi.y * ratio)) << 16;
    }
    *at = make_uint2(c[0], c[1]);
  }
}

// The page's scale for new tokens with this largest element, and whether it is
// to be written; ratio != 1: held codes are to be multiplied by it.
struct NewScale {
  float scale, ratio;
  bool write;
};
__device__ __forceinline__ NewScale new_scale(const QuantStoreParams &p, float amax, int held, float old, bool report) {
  NewScale n{scale_for(amax), 1.f, true};
  if (held > 0) {
    if (!good_scale(old)) {
      if (report) raise_deverr(p.error_word, YL_DEVERR_SCALE);
    } else if (n.scale > old) {
      n.ratio = old / n.scale;
    } else {
      n.scale = old;
      n.write = false;
    }
  }
  return n;
}

// This lane's part of the first row of a page's new tokens in a plane.
template <int D>
__device__ __forceinline__ const char *row_of(const QuantStoreParams &p, int64_t row0, int plane, int h, int lane) {
  const int kv = plane & 1, layer = plane >> 1;
  return p.x[kv] + layer * p.layer_stride[kv] + row0 * p.row_stride[kv] + static_cast<int64_t>(h) * (D * 2) +
         lane % (D / 8) * 16;
}

// PB planes of one page at once, each with at most RB new tokens, which x holds.
template <typename T, int D, int PB, int RB>
__device__ __forceinline__ void store_planes(const QuantStoreParams &p, const Touched &pg, int plane0, int count,
                                             int head, int lane, uint4 (&x)[PB][RB]) {
  constexpr int LPR = D / 8;
  const int sub = lane % LPR;
  const bool active = head < p.pool.num_heads;
  const int h = active ? head : 0;
  float old[PB];
  const char *src[PB];
#pragma unroll
  for (int b = 0; b < PB; ++b) {
    const int plane = plane0 + b, kv = plane & 1, layer = plane >> 1;
    src[b] = row_of<D>(p, pg.row0, plane, h, lane);
    old[b] = 0.f;
    if (b < count && active && pg.held > 0)
      old[b] = p.pool.scale[kv][layer * p.pool.scale_layer_stride + pg.page * p.pool.scale_page_stride +
                                h * p.pool.scale_head_stride];
  }
  __syncwarp();  // every lane has the old scales
#pragma unroll
  for (int b = 0; b < PB; ++b) {
    const int plane = plane0 + b, kv = plane & 1, layer = plane >> 1;
    const int64_t stride = p.row_stride[kv];
    uint32_t m = 0;
    if (b < count && active) {
#pragma unroll
      for (int r = 0; r < RB; ++r)
        if (r < pg.count) m = abs_max8(m, x[b][r]);
    }
#pragma unroll
    for (int d = LPR / 2; d > 0; d >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
    m = max(m & 0xffffu, m >> 16);
    float amax = T::unpack(m).x;
    // an infinity or NaN somewhere in the warp's rows: the finite maximum, the slow way
    if (__any_sync(0xffffffffu, m >= T::kInf)) {
      float f = 0.f;
      if (b < count && active)
        for (int r = 0; r < pg.count; ++r)
          f = finite_abs_max8<T>(f, __ldg(reinterpret_cast<const uint4 *>(src[b] + r * stride)));
#pragma unroll
      for (int d = LPR / 2; d > 0; d >>= 1) f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, d));
      if (m >= T::kInf && sub == 0) raise_deverr(p.error_word, YL_DEVERR_NONFINITE);
      amax = f;
    }
    if (b < count && active) {
      uint8_t *dst = p.pool.codes[kv] + layer * p.pool.layer_stride + pg.page * p.pool.page_stride +
                     h * p.pool.head_stride + sub * 8;
      float *sc = p.pool.scale[kv] + layer * p.pool.scale_layer_stride + pg.page * p.pool.scale_page_stride +
                  h * p.pool.scale_head_stride;
      const NewScale n = new_scale(p, amax, pg.held, old[b], sub == 0);
      if (n.ratio != 1.f) requantise(dst, p.pool.slot_stride, 0, pg.held, 1, n.ratio);
      if (n.write && sub == 0) *sc = n.scale;
      const float inv = 1.f / n.scale;  // exact for a power of two
      dst += pg.held * p.pool.slot_stride;
#pragma unroll
      for (int r = 0; r < RB; ++r)
        if (r < pg.count) *reinterpret_cast<uint2 *>(dst + r * p.pool.slot_stride) = quantise8<T>(x[b][r], inv);
    }
  }
}

// A page of several new tokens in a batch of mostly one each: rows read twice.
template <typename T, int D>
__device__ __noinline__ void store_rows_twice(const QuantStoreParams &p, const Touched &pg, int plane, int head, int lane) {
  constexpr int LPR = D / 8;
  const int kv = plane & 1, layer = plane >> 1, sub = lane % LPR;
  const bool active = head < p.pool.num_heads;
  const int h = active ? head : 0;
  const int64_t stride = p.row_stride[kv];
  const char *src = row_of<D>(p, pg.row0, plane, h, lane);
  float *sc = p.pool.scale[kv] + layer * p.pool.scale_layer_stride + pg.page * p.pool.scale_page_stride +
              h * p.pool.scale_head_stride;
  const float old = active && pg.held > 0 ? *sc : 0.f;
  float amax = 0.f;
  bool bad = false;
  if (active)
    for (int r = 0; r < pg.count; ++r) {
      const uint4 w = __ldg(reinterpret_cast<const uint4 *>(src + r * stride));
      const uint32_t m = abs_max8(0, w);
      bad |= max(m & 0xffffu, m >> 16) >= T::kInf;
      amax = finite_abs_max8<T>(amax, w);
    }
#pragma unroll
  for (int d = LPR / 2; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, d));
  if (bad) raise_deverr(p.error_word, YL_DEVERR_NONFINITE);
  __syncwarp();  // every lane has the old scale
  if (!active) return;
  uint8_t *dst = p.pool.codes[kv] + layer * p.pool.layer_stride + pg.page * p.pool.page_stride + h * p.pool.head_stride +
                 sub * 8;
  const NewScale n = new_scale(p, amax, pg.held, old, sub == 0);
  if (n.ratio != 1.f) requantise(dst, p.pool.slot_stride, 0, pg.held, 1, n.ratio);
  if (n.write && sub == 0) *sc = n.scale;
  const float inv = 1.f / n.scale;  // exact for a power of two
  dst += pg.held * p.pool.slot_stride;
  for (int r = 0; r < pg.count; ++r)
    *reinterpret_cast<uint2 *>(dst + r * p.pool.slot_stride) =
        quantise8<T>(__ldg(reinterpret_cast<const uint4 *>(src + r * stride)), inv);
}

// How a page's new tokens are dealt out.  kByToken (batches of mostly one new
// token a sequence, and pages of one): a warp's first rows are known before its
// page is, so they are loaded in front of the look-ups, eight planes at once.
// kByWarp: up to 16 rows of a page by a warp.  kByBlock (pages of more than 16
// tokens): four warps share a page, up to 64 rows in registers, and exchange
// their maxima; of longer pages the rows are read twice.  They are kernels of
// their own, since the registers of one would cost the other's warps in flight.
// Both sides of each rule, 32 layers of 8 heads of 128: 256 sequences of one token
// by token 22.6 us, by warp 29.4; 64 prompts in pages of 16 by warp 269 us, by
// block 659; pages of 8 by warp 351, by block 1,208; pages of 64 by block 274,
// by warp 528.
enum StoreMode { kByToken, kByWarp, kByBlock };

template <typename T, int D>
__device__ __forceinline__ void store_by_block(const QuantStoreParams &p, const Touched &pg, int first, int end, int head,
                                               int lane) {
  constexpr int LPR = D / 8, RPW = 32 / LPR, TEAM = kStoreThreads / 32, SLAB = 16 * TEAM;
  __shared__ uint32_t bits[2][TEAM][RPW];
  __shared__ float finite[TEAM][RPW];
  const int warp = threadIdx.x >> 5, sub = lane % LPR, group = lane / LPR;
  const bool active = head < p.pool.num_heads;
  const int h = active ? head : 0;
  for (int pl = first; pl < end; ++pl) {
    const int kv = pl & 1, layer = pl >> 1, par = pl & 1;
    const int64_t stride = p.row_stride[kv];
    const char *src = row_of<D>(p, pg.row0, pl, h, lane);
    float *sc = p.pool.scale[kv] + layer * p.pool.scale_layer_stride + pg.page * p.pool.scale_page_stride +
                h * p.pool.scale_head_stride;
    const float old = active && pg.held > 0 ? *sc : 0.f;
    uint4 x[16];
    auto load = [&](int slab) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = slab + r * TEAM + warp;
        x[r] = make_uint4(0, 0, 0, 0);
        if (row < pg.count && active) x[r] = __ldg(reinterpret_cast<const uint4 *>(src + row * stride));
      }
    };
    uint32_t m = 0;
    for (int slab = 0; slab < pg.count; slab += SLAB) {
      load(slab);
#pragma unroll
      for (int r = 0; r < 16; ++r) m = abs_max8(m, x[r]);
    }
#pragma unroll
    for (int d = LPR / 2; d > 0; d >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, d));
    if (sub == 0) bits[par][warp][group] = max(m & 0xffffu, m >> 16);
    // (the barrier also ends the reading of a held scale, which is written below,
    // and of bits two planes back)
    __syncthreads();
    m = bits[par][0][group];
#pragma unroll
    for (int w = 1; w < TEAM; ++w) m = max(m, bits[par][w][group]);
    float amax = T::unpack(m).x;
    if (__syncthreads_or(m >= T::kInf)) {  // an infinity or NaN: the finite maximum, the slow way
      float f = 0.f;
      if (active)
        for (int row = warp; row < pg.count; row += TEAM)
          f = finite_abs_max8<T>(f, __ldg(reinterpret_cast<const uint4 *>(src + row * stride)));
#pragma unroll
      for (int d = LPR / 2; d > 0; d >>= 1) f = fmaxf(f, __shfl_xor_sync(0xffffffffu, f, d));
      if (sub == 0) finite[warp][group] = f;
      __syncthreads();
      amax = finite[0][group];
#pragma unroll
      for (int w = 1; w < TEAM; ++w) amax = fmaxf(amax, finite[w][group]);
      __syncthreads();
      if (m >= T::kInf && sub == 0 && warp == 0) raise_deverr(p.error_word, YL_DEVERR_NONFINITE);
    }
    if (!active) continue;
    uint8_t *dst = p.pool.codes[kv] + layer * p.pool.layer_stride + pg.page * p.pool.page_stride + h * p.pool.head_stride +
                   sub * 8;
    const NewScale n = new_scale(p, amax, pg.held, old, sub == 0 && warp == 0);
    if (n.ratio != 1.f) requantise(dst, p.pool.slot_stride, warp, pg.held, TEAM, n.ratio);
    if (n.write && sub == 0 && warp == 0) *sc = n.scale;
    const float inv = 1.f / n.scale;  // exact for a power of two
    dst += pg.held * p.pool.slot_stride;
    for (int slab = 0; slab < pg.count; slab += SLAB) {
      if (pg.count > SLAB) load(slab);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = slab + r * TEAM + warp;
        if (row < pg.count) *reinterpret_cast<uint2 *>(dst + row * p.pool.slot_stride) = quantise8<T>(x[r], inv);
      }
    }
  }
}

template <typename T, int D, StoreMode MODE>
__global__ void __launch_bounds__(kStoreThreads, MODE == kByToken ? 7 : 4)
    quant_store_kernel(const __grid_constant__ QuantStoreParams p) {
  constexpr int RPW = 32 / (D / 8);  // heads a warp takes at once
  constexpr int PB = 8;              // planes at once, by token
  const int lane = threadIdx.x & 31;
  const uint32_t unit = MODE == kByBlock ? blockIdx.x : blockIdx.x * (kStoreThreads / 32) + (threadIdx.x >> 5);
  pdl_wait();  // rows and page arrays may be written by the kernel just before this one
  const uint32_t part = unit % p.chunks, rest = unit / p.chunks;
  const uint32_t cand = rest % p.cands, run = rest / p.cands;
  if (run >= p.runs) return;
  const int first = run * p.planes_per_run;
  const int end = min(first + static_cast<int>(p.planes_per_run), p.planes);
  const bool report = part == 0 && run == 0 && lane == 0 && (MODE != kByBlock || threadIdx.x == 0);
  const int head = static_cast<int>(part) * RPW + lane / (D / 8);
  if (MODE == kByToken) {
    uint4 x[PB][1];
    auto load = [&](int plane0) {
#pragma unroll
      for (int b = 0; b < PB; ++b)
        if (plane0 + b < end && head < p.pool.num_heads)
          x[b][0] = __ldg(reinterpret_cast<const uint4 *>(row_of<D>(p, cand, plane0 + b, head, lane)));
    };
    load(first);
    const Touched pg = find_page<true>(p, cand, lane, report);
    if (pg.count == 0) return;
    if (pg.count == 1) {  // then it is row `cand`
      for (int pl = first; pl < end; pl += PB) {
        if (pl > first) load(pl);
        store_planes<T, D, PB, 1>(p, pg, pl, end - pl, head, lane, x);
      }
    } else {
      for (int pl = first; pl < end; ++pl) store_rows_twice<T, D>(p, pg, pl, head, lane);
    }
  } else {
    const Touched pg = find_page<false>(p, cand, lane, report);
    if (pg.count == 0) return;
    if (MODE == kByBlock) {
      store_by_block<T, D>(p, pg, first, end, head, lane);
    } else {
      for (int pl = first; pl < end; ++pl) {
        uint4 x[1][16];
        const bool active = head < p.pool.num_heads;
        const char *src = row_of<D>(p, pg.row0, pl, active ? head : 0, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (r < pg.count && active) x[0][r] = __ldg(reinterpret_cast<const uint4 *>(src + r * p.row_stride[pl & 1]));
        store_planes<T, D, 1, 16>(p, pg, pl, 1, head, lane, x);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Load.  A lane group of head_dim / 16 lanes owns a row (plane, token, head):
// one 16-byte load of codes, two 16-byte stores per lane, kLoadRows rows of a
// group in flight.
// ---------------------------------------------------------------------------
struct QuantLoadParams {
  QuantPool pool;
  char *out[2];
  int64_t row_stride[2], layer_stride[2];
  const void *slots;
  uint32_t *error_word;
  int64_t num_slots;
  uint32_t rows;  // planes * tokens * heads
  FastDiv by_heads, by_tokens, by_page;
};

constexpr int kLoadThreads = 256;
constexpr int kLoadRows = 4;

template <typename T, int D, typename Slot, bool WIDE>
__global__ void __launch_bounds__(kLoadThreads) quant_load_kernel(const __grid_constant__ QuantLoadParams p) {
  constexpr int LPR = D / 16;
  constexpr int GROUPS = kLoadThreads / LPR;
  const int sub = threadIdx.x % LPR;
  const Slot *slots = static_cast<const Slot *>(p.slots);
  pdl_wait();  // the pool and the slots may be written by the kernel just before this one
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * GROUPS * kLoadRows;
  for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * GROUPS * kLoadRows + threadIdx.x / LPR; base < p.rows;
       base += step) {
    uint4 w[kLoadRows];
    float scale[kLoadRows];
    char *dst[kLoadRows];
#pragma unroll
    for (int u = 0; u < kLoadRows; ++u) {
      const uint64_t r64 = base + static_cast<uint64_t>(u) * GROUPS;
      w[u] = make_uint4(0, 0, 0, 0);
      scale[u] = 0.f;
      dst[u] = nullptr;
      if (r64 >= p.rows) continue;
      const uint32_t r = static_cast<uint32_t>(r64);
      const uint32_t pt = p.by_heads.div(r), head = r - pt * p.by_heads.d;
      const uint32_t plane = p.by_tokens.div(pt), token = pt - plane * p.by_tokens.d;
      const int kv = plane & 1;
      const int64_t layer = plane >> 1;
      dst[u] = p.out[kv] + layer * p.layer_stride[kv] + token * p.row_stride[kv] + static_cast<int64_t>(head) * (D * 2) +
               sub * 32;
      const int64_t slot = __ldg(slots + token);
      if (slot < 0 || slot >= p.num_slots) {
        if (slot != -1 && sub == 0 && plane == 0 && head == 0) raise_deverr(p.error_word, YL_DEVERR_SLOT_RANGE);
        continue;
      }
      const uint32_t page = p.by_page.div(static_cast<uint32_t>(slot));
      const uint32_t off = static_cast<uint32_t>(slot) - page * p.by_page.d;
      scale[u] = __ldg(p.pool.scale[kv] + layer * p.pool.scale_layer_stride + page * p.pool.scale_page_stride +
                       head * p.pool.scale_head_stride);
      w[u] = __ldg(reinterpret_cast<const uint4 *>(p.pool.codes[kv] + layer * p.pool.layer_stride +
                                                   page * p.pool.page_stride + off * p.pool.slot_stride +
                                                   head * p.pool.head_stride + sub * 16));
    }
#pragma unroll
    for (int u = 0; u < kLoadRows; ++u) {
      if (dst[u] == nullptr) continue;
      const uint32_t v[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
      uint32_t o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 f =
            half2_bits_to_float2(e4m3x2_to_half2(static_cast<uint16_t>(i & 1 ? v[i / 2] >> 16 : v[i / 2] & 0xffffu)));
        // past T's range: T's largest; NaN passes both comparisons unchanged
        float a = f.x * scale[u], b = f.y * scale[u];
        a = a > T::kMax ? T::kMax : a < -T::kMax ? -T::kMax : a;
        b = b > T::kMax ? T::kMax : b < -T::kMax ? -T::kMax : b;
        o[i] = T::pack(a, b);
      }
      if (WIDE) {
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst[u]), "r"(o[0]), "r"(o[1]), "r"(o[2]),
                     "r"(o[3]), "r"(o[4]), "r"(o[5]), "r"(o[6]), "r"(o[7])
                     : "memory");
      } else {
        reinterpret_cast<uint4 *>(dst[u])[0] = make_uint4(o[0], o[1], o[2], o[3]);
        reinterpret_cast<uint4 *>(dst[u])[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_pool(const yl_quant_pool &q, int align, const char *who, QuantPool &out) {
  auto bad = [&](int status, const char *what, long long a = 0) {
    char buf[200];
    std::snprintf(buf, sizeof(buf), "%s: %s", who, what);
    return fail(status, buf, a);
  };
  if (q.num_layers < 1) return bad(YL_ERR_BAD_SIZE, "num_layers=%lld < 1", q.num_layers);
  if (q.page_size < 1) return bad(YL_ERR_BAD_SIZE, "page_size=%lld < 1", q.page_size);
  if (q.num_heads < 1) return bad(YL_ERR_BAD_SIZE, "num_heads=%lld < 1", q.num_heads);
  if (q.num_pages < 1) return bad(YL_ERR_BAD_SIZE, "num_pages=%lld < 1", q.num_pages);
  if (q.num_layers >= 1 << 24 || q.num_heads >= 1 << 24)
    return bad(YL_ERR_UNSUPPORTED, "num_layers=%lld and num_heads must be below 2^24", q.num_layers);
  if (q.head_dim != 64 && q.head_dim != 128 && q.head_dim != 256)
    return bad(YL_ERR_UNSUPPORTED, "head_dim=%lld must be 64, 128 or 256", q.head_dim);
  if (q.num_pages >= (1ll << 31) || q.num_pages * q.page_size >= (1ll << 31))
    return bad(YL_ERR_UNSUPPORTED, "num_pages * page_size=%lld must be below 2^31", q.num_pages);
  if (!q.k_codes || !q.v_codes || !q.k_scale || !q.v_scale)
    return bad(YL_ERR_NULL_ARG, "k_codes, v_codes, k_scale and v_scale must be non-NULL");
  if (q.slot_stride < q.head_dim || q.head_stride < q.head_dim || q.page_stride < q.head_dim || q.layer_stride < 0)
    return bad(YL_ERR_BAD_SIZE, "code strides must be at least head_dim=%lld", q.head_dim);
  if (q.scale_page_stride < 1 || q.scale_head_stride < 1 || q.scale_layer_stride < 0)
    return bad(YL_ERR_BAD_SIZE, "scale strides must be positive");
  const uintptr_t bits = reinterpret_cast<uintptr_t>(q.k_codes) | reinterpret_cast<uintptr_t>(q.v_codes) |
                         static_cast<uintptr_t>(q.slot_stride) | static_cast<uintptr_t>(q.head_stride) |
                         static_cast<uintptr_t>(q.page_stride) |
                         static_cast<uintptr_t>(q.num_layers > 1 ? q.layer_stride : 0);
  if (bits & static_cast<uintptr_t>(align - 1))
    return bad(YL_ERR_ALIGNMENT, "codes and their strides must be multiples of %lld bytes", align);
  if ((reinterpret_cast<uintptr_t>(q.k_scale) | reinterpret_cast<uintptr_t>(q.v_scale)) & 3u)
    return bad(YL_ERR_ALIGNMENT, "scales must be 4-byte aligned");
  out = QuantPool{{static_cast<uint8_t *>(q.k_codes), static_cast<uint8_t *>(q.v_codes)},
                  {q.k_scale, q.v_scale},
                  q.num_layers > 1 ? q.layer_stride : 0,
                  q.page_stride, q.slot_stride, q.head_stride,
                  q.num_layers > 1 ? q.scale_layer_stride : 0,
                  q.scale_page_stride, q.scale_head_stride,
                  static_cast<int32_t>(q.num_pages), q.page_size, q.num_heads};
  return YL_OK;
}

int check_rows(const void *k, const void *v, int64_t ks, int64_t vs, int64_t kl, int64_t vl, const yl_quant_pool &q,
               const char *who) {
  auto bad = [&](int status, const char *what, long long a = 0) {
    char buf[200];
    std::snprintf(buf, sizeof(buf), "%s: %s", who, what);
    return fail(status, buf, a);
  };
  const int64_t row = static_cast<int64_t>(q.num_heads) * q.head_dim * 2;
  if (ks < row || vs < row) return bad(YL_ERR_BAD_SIZE, "row strides must be at least the row's %lld bytes", row);
  if (q.num_layers > 1 && (kl < 0 || vl < 0)) return bad(YL_ERR_BAD_SIZE, "layer strides must not be negative");
  uintptr_t bits = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | static_cast<uintptr_t>(ks) |
                   static_cast<uintptr_t>(vs);
  if (q.num_layers > 1) bits |= static_cast<uintptr_t>(kl) | static_cast<uintptr_t>(vl);
  if (bits & 15u) return bad(YL_ERR_ALIGNMENT, "row pointers and strides must be multiples of 16 bytes");
  return YL_OK;
}

template <typename F>
auto pick_type_dim(int dtype, int dim, F f) {
  if (dtype == YL_DTYPE_BF16) {
    if (dim == 64) return f(Bf16{}, std::integral_constant<int, 64>{});
    if (dim == 128) return f(Bf16{}, std::integral_constant<int, 128>{});
    return f(Bf16{}, std::integral_constant<int, 256>{});
  }
  if (dim == 64) return f(Fp16{}, std::integral_constant<int, 64>{});
  if (dim == 128) return f(Fp16{}, std::integral_constant<int, 128>{});
  return f(Fp16{}, std::integral_constant<int, 256>{});
}

}  // namespace
}  // namespace ylk

extern "C" int yl_kv_quant_store(const yl_quant_store_args *a, cudaStream_t stream) {
  using namespace ylk;
  clear_last_error();
  const char *who = "yl_kv_quant_store";
  if (a == nullptr) return fail(YL_ERR_NULL_ARG, "yl_kv_quant_store: args is NULL");
  if (a->batch_size < 0) return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_store: batch_size=%lld < 0", a->batch_size);
  if (a->num_tokens < 0) return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_store: num_tokens=%lld < 0", a->num_tokens);
  if (a->kv_indices_capacity < 0)
    return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_store: kv_indices_capacity=%lld < 0", a->kv_indices_capacity);
  if (a->dtype != YL_DTYPE_BF16 && a->dtype != YL_DTYPE_F16)
    return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_store: dtype=%lld unknown", a->dtype);
  if (a->batch_size == 0 || a->num_tokens == 0) return YL_OK;
  QuantStoreParams p;
  int rc = check_pool(a->pool, 8, who, p.pool);
  if (rc != YL_OK) return rc;
  if (!a->k || !a->v || !a->kv_indptr || !a->kv_last_page_len || !a->qo_indptr ||
      (!a->kv_indices && a->kv_indices_capacity > 0))
    return fail(YL_ERR_NULL_ARG, "yl_kv_quant_store: k, v and the page arrays must be non-NULL");
  if ((reinterpret_cast<uintptr_t>(a->kv_indptr) | reinterpret_cast<uintptr_t>(a->kv_indices) |
       reinterpret_cast<uintptr_t>(a->kv_last_page_len) | reinterpret_cast<uintptr_t>(a->qo_indptr) |
       reinterpret_cast<uintptr_t>(a->error_word)) & 3u)
    return fail(YL_ERR_ALIGNMENT, "yl_kv_quant_store: page arrays and error_word must be 4-byte aligned");
  rc = check_rows(a->k, a->v, a->k_row_stride, a->v_row_stride, a->k_layer_stride, a->v_layer_stride, a->pool, who);
  if (rc != YL_OK) return rc;
  if (a->pool.num_layers > 1 && (a->pool.layer_stride < 1 || a->pool.scale_layer_stride < 1))
    return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_store: the pool's layers must lie apart");
  if (a->num_tokens >= (1ll << 31))
    return fail(YL_ERR_UNSUPPORTED, "yl_kv_quant_store: num_tokens=%lld must be below 2^31", a->num_tokens);
  p.x[0] = static_cast<const char *>(a->k);
  p.x[1] = static_cast<const char *>(a->v);
  p.row_stride[0] = a->k_row_stride;
  p.row_stride[1] = a->v_row_stride;
  p.layer_stride[0] = a->pool.num_layers > 1 ? a->k_layer_stride : 0;
  p.layer_stride[1] = a->pool.num_layers > 1 ? a->v_layer_stride : 0;
  p.kv_indptr = a->kv_indptr;
  p.kv_indices = a->kv_indices;
  p.last_len = a->kv_last_page_len;
  p.qo_indptr = a->qo_indptr;
  p.indices_cap = a->kv_indices_capacity;
  p.num_tokens = a->num_tokens;
  p.error_word = a->error_word;
  p.batch = a->batch_size;
  p.planes = 2 * a->pool.num_layers;
  const int64_t by_page = a->num_tokens / a->pool.page_size + 2ll * a->batch_size;
  const bool by_token = a->num_tokens <= by_page;
  p.cands = static_cast<uint32_t>(by_token ? a->num_tokens : by_page);
  const StoreMode mode = by_token ? kByToken : a->pool.page_size <= 16 ? kByWarp : kByBlock;
  const int heads_per_warp = 256 / a->pool.head_dim;
  p.chunks = static_cast<uint32_t>((a->pool.num_heads + heads_per_warp - 1) / heads_per_warp);
  const uint64_t resident = static_cast<uint64_t>(sm_count()) * (mode == kByToken ? 28 : 16);  // warps
  // By token a wave of resident warps; by page, where a warp's work is longer, up
  // to four waves.
  const uint64_t items = static_cast<uint64_t>(p.cands) * p.chunks * (mode == kByBlock ? 4 : 1);
  const uint64_t runs = std::min<uint64_t>(
      std::max<uint64_t>(mode == kByToken ? resident / items : (4 * resident + items - 1) / items, 1), p.planes);
  p.planes_per_run = static_cast<uint32_t>((p.planes + runs - 1) / runs);
  p.runs = (p.planes + p.planes_per_run - 1) / p.planes_per_run;
  const uint64_t units = static_cast<uint64_t>(p.cands) * p.chunks * p.runs;
  if (units >= (1ull << 31))
    return fail(YL_ERR_UNSUPPORTED, "yl_kv_quant_store: %lld pages and heads in one call", (long long)units);
  const unsigned grid =
      static_cast<unsigned>(mode == kByBlock ? units : (units + kStoreThreads / 32 - 1) / (kStoreThreads / 32));
  return pick_type_dim(a->dtype, a->pool.head_dim, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    auto fn = mode == kByToken  ? quant_store_kernel<T, D, kByToken>
              : mode == kByWarp ? quant_store_kernel<T, D, kByWarp>
                                : quant_store_kernel<T, D, kByBlock>;
    return launch_dependent(fn, dim3(grid), dim3(kStoreThreads), 0, stream, "yl_kv_quant_store launch", p);
  });
}

extern "C" int yl_kv_quant_load(const yl_quant_load_args *a, cudaStream_t stream) {
  using namespace ylk;
  clear_last_error();
  const char *who = "yl_kv_quant_load";
  if (a == nullptr) return fail(YL_ERR_NULL_ARG, "yl_kv_quant_load: args is NULL");
  if (a->num_tokens < 0) return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_load: num_tokens=%lld < 0", a->num_tokens);
  if (a->slot_is_int64 != 0 && a->slot_is_int64 != 1)
    return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_load: slot_is_int64=%lld must be 0 or 1", a->slot_is_int64);
  if (a->dtype != YL_DTYPE_BF16 && a->dtype != YL_DTYPE_F16)
    return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_load: dtype=%lld unknown", a->dtype);
  if (a->num_tokens == 0) return YL_OK;
  QuantLoadParams p;
  int rc = check_pool(a->pool, 16, who, p.pool);
  if (rc != YL_OK) return rc;
  if (!a->k_out || !a->v_out || !a->slots)
    return fail(YL_ERR_NULL_ARG, "yl_kv_quant_load: k_out, v_out and slots must be non-NULL");
  rc = check_rows(a->k_out, a->v_out, a->k_row_stride, a->v_row_stride, a->k_layer_stride, a->v_layer_stride, a->pool,
                  who);
  if (rc != YL_OK) return rc;
  if (a->pool.num_layers > 1 && (a->k_layer_stride < 1 || a->v_layer_stride < 1))
    return fail(YL_ERR_BAD_SIZE, "yl_kv_quant_load: the layers of k_out and v_out must lie apart");
  const uintptr_t ib = a->slot_is_int64 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(a->slots) & (ib - 1))
    return fail(YL_ERR_ALIGNMENT, "yl_kv_quant_load: slots pointer is not %lld-byte aligned", (long long)ib);
  if (reinterpret_cast<uintptr_t>(a->error_word) & 3u)
    return fail(YL_ERR_ALIGNMENT, "yl_kv_quant_load: error_word must be 4-byte aligned");
  const int64_t planes = 2ll * a->pool.num_layers;
  if (a->num_tokens >= (1ll << 31) / planes / a->pool.num_heads)
    return fail(YL_ERR_UNSUPPORTED, "yl_kv_quant_load: num_tokens=%lld times layers and heads passes 2^31",
                a->num_tokens);
  p.out[0] = static_cast<char *>(a->k_out);
  p.out[1] = static_cast<char *>(a->v_out);
  p.row_stride[0] = a->k_row_stride;
  p.row_stride[1] = a->v_row_stride;
  p.layer_stride[0] = a->pool.num_layers > 1 ? a->k_layer_stride : 0;
  p.layer_stride[1] = a->pool.num_layers > 1 ? a->v_layer_stride : 0;
  p.slots = a->slots;
  p.error_word = a->error_word;
  p.num_slots = a->pool.num_pages * a->pool.page_size;
  p.rows = static_cast<uint32_t>(planes * a->num_tokens * a->pool.num_heads);
  p.by_heads = FastDiv(static_cast<uint32_t>(a->pool.num_heads));
  p.by_tokens = FastDiv(static_cast<uint32_t>(a->num_tokens));
  p.by_page = FastDiv(static_cast<uint32_t>(a->pool.page_size));
  return pick_type_dim(a->dtype, a->pool.head_dim, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    // 32-byte stores where rows and strides allow them
    const bool wide = ((reinterpret_cast<uintptr_t>(a->k_out) | reinterpret_cast<uintptr_t>(a->v_out) |
                        static_cast<uintptr_t>(p.row_stride[0] | p.row_stride[1] | p.layer_stride[0] | p.layer_stride[1])) &
                       31u) == 0;
    auto fn = a->slot_is_int64 ? (wide ? quant_load_kernel<T, D, int64_t, true> : quant_load_kernel<T, D, int64_t, false>)
                               : (wide ? quant_load_kernel<T, D, int32_t, true> : quant_load_kernel<T, D, int32_t, false>);
    const uint64_t per_block = static_cast<uint64_t>(kLoadThreads / (D / 16)) * kLoadRows;
    const uint64_t want = (p.rows + per_block - 1) / per_block;
    const uint64_t cap = static_cast<uint64_t>(sm_count()) * 8;
    return launch_dependent(fn, dim3(static_cast<unsigned>(std::min(want, cap))), dim3(kLoadThreads), 0, stream,
                            "yl_kv_quant_load launch", p);
  });
}
