// Paged attention of sequences with few new tokens (decode), for sm_100a.
//
// The keys and values are read once and the arithmetic is small, so HBM bounds
// it: 2 * visible tokens * head_dim * item bytes per KV head.  What the design
// is for is keeping every SM's loads in flight to the end:
//
// * The batch's work is one line of units, a unit being a tile of 64 visible
//   tokens of one (sequence, KV head, 16 query rows); the query rows of a unit
//   are the new tokens times the heads of the group.  Each CTA takes an equal
//   run of that line, whatever the lengths of the sequences; each finds its
//   place by scanning the batch itself (a few KB), so a call needs no plan.
//   A (sequence, head) whose units fall in several CTAs leaves its parts in the
//   workspace, and a second kernel joins them, in a fixed order.
// * One warp of a CTA only issues loads: it walks the units, looks up pages one
//   unit ahead, and fills a ring of stages with 16-byte asynchronous copies,
//   across the ends of sequences.  Tokens that no query sees are zero-filled,
//   not read.
// * Four warps compute, 16 tokens of a stage each, with their own running
//   maximum, sum and accumulator (online softmax); the four are joined when a
//   (sequence, head) ends.  Products are m16n8k16 matrix instructions on 16
//   query rows: at 4 to 16 rows these tiles cost less issue than the loads cost
//   bandwidth, which a 128-row tensor tile would waste on padding.
// * An 8-bit pool is multiplied in fp16: every e4m3 value is exact there.  bf16
//   queries are first brought into fp16's range by a power of two per row,
//   exact for all elements within 2^-24 of the row's largest.  The contraction
//   order of q.k is free, so a lane takes 4 neighbouring codes as its part of a
//   k-step and K needs no transposition; the codes of two tokens of V are
//   interleaved by byte permutes before conversion.  K's scale multiplies the
//   scores; V's scale, relative to the largest seen so far, multiplies the
//   weights before they are rounded.  Weights are kept times 2^15, which puts
//   fp16's smallest numbers 2^-39 below the largest weight.
// * All sums, maxima and accumulators are fp32; weights are rounded once, to
//   fp16 (8-bit and fp16 pools) or bf16 (bf16 pools), as the matrix
//   instructions take them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <map>
#include <mutex>
#include <tuple>

#include "attend_device.cuh"
#include "tma.cuh"

namespace ylk {
namespace {

constexpr int kTile = 64;     // tokens of a unit
constexpr int kConsumers = 4; // warps that compute, kTile / 4 tokens each
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kRows = 16;     // query rows of a unit
// A CTA's run is at least this many units, so that a short sequence is not cut
// into parts whose joining costs more than they save.
constexpr int kMinRun = 2;

// Unit descriptor in a stage, written by the loading warp.
struct UnitInfo {
  uint32_t valid[2];  // tokens of the tile that some query sees, with a good page
  int base;           // position of the tile's first token
  int flags;          // kFirst | kLast | kWhole | kRagged
  int pos0;           // position of the sequence's first query
  int row0;           // first query row of the unit: token * group + head of the group
  int rows;           // query rows of the sequence and KV head
  int q0;             // first row of q and o of the sequence
  int head;           // KV head
  int part;           // slot in the workspace of an unfinished result
};
constexpr int kFirst = 1;   // first unit of a (sequence, head, rows) in this CTA
constexpr int kLast = 2;    // last one
constexpr int kWhole = 4;   // with kLast: this CTA has all of its units
constexpr int kRagged = 8;  // some query does not see some valid token

template <int D, bool Q8>
struct Layout {
  static constexpr int kItem = Q8 ? 1 : 2;
  static constexpr int kRow = D * kItem;            // bytes of a token's head row
  static constexpr int kChunks = kRow / 16;         // 16-byte chunks of it
  static constexpr int kKV = kTile * kRow;          // bytes of K (or V) in a stage
  static constexpr int kQ = kRows * D * 2;
  static constexpr int kScales = Q8 ? 2 * kTile * 4 : 0;
  static constexpr int kStage = 2 * kKV + kQ + kScales + 64;
  static constexpr int kMerge = 2 * kRows * D * 4;  // two warps' accumulators
  // two CTAs per SM where a stage is small enough for three of them each
  static constexpr int kCtas = kStage * 3 + kMerge + 1024 <= 113 * 1024 ? 2 : 1;
  static constexpr int kBudget = (kCtas == 2 ? 113 : 226) * 1024 - kMerge - 1024;
  static constexpr int kStages = kBudget / kStage > 8 ? 8 : kBudget / kStage;
  static constexpr int kSmem = kStages * kStage + kMerge + 1024;
  static_assert(kStages >= 2, "a ring needs two stages");
};

// Position of 16-byte chunk c of token row r in a tile.  The chunks of a
// 128-byte line are permuted so that both the 8 lanes that read one chunk
// column of K and the 8 that read neighbouring tokens of V meet all banks.
template <int D, bool Q8>
__device__ __forceinline__ int chunk_at(int r, int c) {
  if (Q8 && D == 64) {  // two rows to a line
    const int line = r >> 1, f = ((line & 1) << 2) | (line & 2);
    return line * 128 + ((((r & 1) * 4 + c) ^ f) << 4);
  }
  const int f = Q8 ? ((((r & 1) ^ ((r >> 2) & 1)) << 2) | (r & 2)) : (r & 7);
  return r * Layout<D, Q8>::kRow + (((c & ~7) | ((c ^ f) & 7)) << 4);
}

template <bool BF>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at));
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t w) { return e4m3x2_to_half2(static_cast<uint16_t>(w)); }
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t w) { return e4m3x2_to_half2(static_cast<uint16_t>(w >> 16)); }

// Zero the 16-bit halves of w that hold an infinity or NaN; bit 0 / 1 of the
// result says which did.
template <bool BF>
__device__ __forceinline__ uint32_t drop_nonfinite(uint32_t &w) {
  constexpr uint32_t inf = BF ? 0x7f80u : 0x7c00u;
  uint32_t bad = 0;
  if ((w & inf) == inf) {
    bad |= 1;
    w &= 0xffff0000u;
  }
  if (((w >> 16) & inf) == inf) {
    bad |= 2;
    w &= 0x0000ffffu;
  }
  return bad;
}

// ---------------------------------------------------------------------------
// The line of units
// ---------------------------------------------------------------------------
struct SeqWork {
  int row_tiles;
  int head_tiles;  // tiles of the first visible positions
  int tiles;       // tiles of one (head, row tile)
  int64_t units;
};

__device__ __forceinline__ SeqWork work_of(const AttnParams &p, const Seq &s) {
  SeqWork w{0, 0, 0, 0};
  const int64_t rows = static_cast<int64_t>(s.fresh) * p.group;
  if (rows == 0 || rows > p.max_rows) return w;
  const Span v = span_of(p, s, 0, s.fresh);
  w.row_tiles = (static_cast<int>(rows) + kRows - 1) / kRows;
  w.head_tiles = (v.head + kTile - 1) / kTile;
  w.tiles = max(1, w.head_tiles + (v.end - v.low + kTile - 1) / kTile);  // nothing visible: one empty tile, zeros
  w.units = static_cast<int64_t>(p.heads) * w.row_tiles * w.tiles;
  return w;
}

struct Place {
  int seq;         // sequence of the run's first unit
  int64_t within;  // that unit, counted from the sequence's first
  int64_t start;   // units before the sequence
  int64_t run, total;
};

// This CTA's place in the line.  Thread t sums the sequences [t m, t m + m).
__device__ __forceinline__ bool find_place(const AttnParams &p, Place &out) {
  __shared__ int64_t warp_sum[kThreads / 32];
  __shared__ Place found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int m = (p.batch + kThreads - 1) / kThreads;
  const int lo = min(tid * m, p.batch), hi = min(lo + m, p.batch);
  int64_t sum = 0;
  for (int i = lo; i < hi; ++i) sum += work_of(p, load_seq(p, i, blockIdx.x == 0)).units;
  int64_t scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += y;
  }
  if (lane == 31) warp_sum[warp] = scan;
  __syncthreads();
  int64_t before = scan - sum, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  const int64_t run = max((total + gridDim.x - 1) / gridDim.x, int64_t(kMinRun));
  const int64_t at = run * blockIdx.x;
  if (at >= total) return false;
  if (before <= at && at < before + sum) {
    int i = lo;
    for (; i < hi - 1; ++i) {
      const int64_t u = work_of(p, load_seq(p, i, false)).units;
      if (at < before + u) break;
      before += u;
    }
    found = Place{i, at - before, before, run, total};
  }
  __syncthreads();
  out = found;
  return true;
}

// ---------------------------------------------------------------------------
// Loading warp
// ---------------------------------------------------------------------------
template <int D, bool Q8>
__device__ void load_units(const AttnParams &p, const Place &place, uint8_t *stages, uint64_t *full, uint64_t *empty) {
  using L = Layout<D, Q8>;
  const int lane = threadIdx.x & 31;
  const int64_t first = place.run * blockIdx.x;
  const int count = static_cast<int>(min(place.run, place.total - first));
  int i = place.seq;
  Seq s = load_seq(p, i, false);
  SeqWork w = work_of(p, s);
  int64_t begin = place.start;  // units before sequence i
  int rt_tile = static_cast<int>(place.within % w.tiles);
  int64_t rest = place.within / w.tiles;
  int rt = static_cast<int>(rest % w.row_tiles);
  int head = static_cast<int>(rest / w.row_tiles);
  Span v = span_of(p, s, 0, s.fresh);

  // page ids of two tokens per lane, looked up one unit ahead
  int base, cnt, page[2];
  auto look_up = [&]() {
    const bool in_head = rt_tile < w.head_tiles;
    const int t = in_head ? rt_tile : rt_tile - w.head_tiles;
    base = (in_head ? 0 : v.low) + t * kTile;
    cnt = min(kTile, (in_head ? v.head : v.end) - base);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t2 = lane + 32 * k;
      page[k] = -1;
      if (t2 < cnt) {
        const int64_t e = static_cast<int64_t>(s.e0) + p.by_page.div(base + t2);
        if (e >= 0 && e < p.indices_cap) {
          page[k] = __ldg(p.kv_indices + e);
          if (page[k] < 0 || page[k] >= p.num_pages) {
            page[k] = -1;
            raise_deverr(p.error_word, YL_DEVERR_PAGE_RANGE);
          }
        } else {
          raise_deverr(p.error_word, YL_DEVERR_INDICES_CAP);
        }
      }
    }
  };
  look_up();
  uint32_t phase = 1;  // a fresh stage counts as consumed
  int stage = 0;
  for (int u = 0; u < count; ++u) {
    uint8_t *st = stages + stage * L::kStage;
    const uint32_t sk = smem_addr(st), sv = sk + L::kKV, sq = sv + L::kKV, ss = sq + L::kQ;
    // this unit's numbers; the look-up of the next one overwrites them
    const int tile = rt_tile, u_base = base, u_cnt = cnt, u_head = head, u_rt = rt;
    const Seq us = s;
    const SeqWork uw = w;
    const int64_t seg = begin + (static_cast<int64_t>(head) * w.row_tiles + rt) * w.tiles;  // its first unit in the line
    int64_t off[2];
    uint32_t valid[2];
    int64_t sc[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int t2 = lane + 32 * k;
      const bool ok = page[k] >= 0;
      const int pos = u_base + t2;
      const int slot = pos - static_cast<int>(p.by_page.div(max(pos, 0))) * p.page_size;
      off[k] = ok ? static_cast<int64_t>(page[k]) * p.page_stride + static_cast<int64_t>(slot) * p.slot_stride +
                        u_head * p.head_stride
                  : 0;
      sc[k] = ok ? static_cast<int64_t>(page[k]) * p.scale_page_stride + u_head * p.scale_head_stride : 0;
      valid[k] = __ballot_sync(0xffffffffu, ok);
    }
    // on to the next unit's look-up, before this one's copies
    if (u + 1 < count) {
      if (++rt_tile == w.tiles) {
        rt_tile = 0;
        if (++rt == w.row_tiles) {
          rt = 0;
          if (++head == p.heads) {
            head = 0;
            begin += w.units;
            do {  // ends: count units remain in the line
              s = load_seq(p, ++i, false);
              w = work_of(p, s);
            } while (w.units == 0 && i + 1 < p.batch);
            v = span_of(p, s, 0, s.fresh);
          }
        }
      }
      look_up();
    }
    if (!mbar_wait_bounded(empty + stage, phase, kBulkWaitLimitNs)) {
      if (lane == 0) raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
      break;
    }
    constexpr int kRowsPer = 32 / L::kChunks;  // rows of one copy instruction
    const int c = lane % L::kChunks;
#pragma unroll 4
    for (int j = 0; j < kTile / kRowsPer; ++j) {
      const int r = j * kRowsPer + lane / L::kChunks;
      const int half = j * kRowsPer / 32;
      const int64_t o = __shfl_sync(0xffffffffu, half ? off[1] : off[0], r & 31) + c * 16;
      const bool ok = ((half ? valid[1] : valid[0]) >> (r & 31)) & 1u;
      const int at = chunk_at<D, Q8>(r, c);
      cp_async16(sk + at, p.kv[0] + o, ok);
      cp_async16(sv + at, p.kv[1] + o, ok);
    }
    if (Q8) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bool ok = (valid[k] >> lane) & 1u;
        cp_async4(ss + (lane + 32 * k) * 4, p.scale[0] + sc[k], ok);
        cp_async4(ss + kTile * 4 + (lane + 32 * k) * 4, p.scale[1] + sc[k], ok);
      }
    }
    const bool is_first = u == 0 || tile == 0;
    const int rows = us.fresh * p.group;
    if (is_first) {
      constexpr int kQChunks = D / 8;
#pragma unroll
      for (int j = 0; j < kRows * kQChunks / 32; ++j) {
        const int n = j * 32 + lane, r = n / kQChunks, qc = n % kQChunks;
        const int row = u_rt * kRows + r;
        const int t = p.by_group.div(row), g = row - t * p.group;
        const int64_t qrow = static_cast<int64_t>(us.q0) + t;
        const bool ok = row < rows && qrow < p.num_tokens;
        const char *src = p.q + (ok ? qrow * p.q_row_stride + (static_cast<int64_t>(u_head) * p.group + g) * p.q_head_stride
                                    : 0) + qc * 16;
        cp_async16(sq + r * D * 2 + (((qc & ~7) | ((qc ^ r) & 7)) << 4), src, ok);
      }
    }
    cp_async_arrive(smem_addr(full + stage));
    if (lane == 0) {
      UnitInfo info;
      info.valid[0] = valid[0];
      info.valid[1] = valid[1];
      info.base = u_base;
      info.pos0 = us.total - us.fresh;
      info.row0 = u_rt * kRows;
      info.rows = rows;
      info.q0 = us.q0;
      info.head = u_head;
      int flags = is_first ? kFirst : 0;
      const bool ends = tile == uw.tiles - 1;
      if (ends || u == count - 1) flags |= kLast;
      if (ends && seg >= first) flags |= kWhole;
      const int last_pos = us.total - 1, end = u_base + u_cnt - 1;
      const bool all = end <= info.pos0 && (p.window == 0 || u_base > last_pos - p.window || end < p.sinks);
      if (us.fresh > 1 && !all) flags |= kRagged;
      info.flags = flags;
      info.part = static_cast<int>(2 * blockIdx.x + (seg >= first ? 1 : 0));
      *reinterpret_cast<UnitInfo *>(st + 2 * L::kKV + L::kQ + L::kScales) = info;
      mbar_arrive(full + stage);
      // where the parts of a result lie that began in an earlier CTA
      if (u == 0) {
        int4 meta = make_int4(0, 0, 0, 0);
        if (seg < first) {
          const int c0 = static_cast<int>(seg / place.run), c1 = static_cast<int>((seg + uw.tiles - 1) / place.run);
          // the first CTA boundary inside it stands for the whole of it
          if (c0 + 1 == static_cast<int>(blockIdx.x)) meta = make_int4(c1 - c0 + 1, us.q0, info.row0 | u_head << 16, rows);
        }
        p.meta[blockIdx.x] = meta;
      }
    }
    if (++stage == L::kStages) {
      stage = 0;
      phase ^= 1;
    }
  }
  cp_async_wait_all();
}

// ---------------------------------------------------------------------------
// Computing warps
// ---------------------------------------------------------------------------
template <typename T, int D, bool Q8>
__device__ void compute_units(const AttnParams &p, const Place &place, uint8_t *stages, uint64_t *full,
                              uint64_t *empty, uint64_t *joined, float *merge) {
  using L = Layout<D, Q8>;
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;  // type of the matrix instructions
  constexpr int KS = D / 16;                                // k-steps of q.k
  constexpr int NT = D / 8;                                 // n-tiles of p.v
  constexpr float kLift = BF ? 0.f : 15.f;                  // weights are kept times 2^kLift
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int64_t first = place.run * blockIdx.x;
  const int count = static_cast<int>(min(place.run, place.total - first));
  uint32_t qf[KS][4];
  float acc[NT][4], m[2], l[2], coef[2], vref = 0.f;
  int stage = 0;
  uint32_t phase = 0, join_phase = 0;
  for (int u = 0; u < count; ++u) {
    uint8_t *st = stages + stage * L::kStage;
    const uint32_t sk = smem_addr(st), sv = sk + L::kKV, sq = sv + L::kKV, ss = sq + L::kQ;
    if (!mbar_wait_bounded(full + stage, phase, kBulkWaitLimitNs)) {
      if (lane == 0) raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
      return;
    }
    const UnitInfo *info = reinterpret_cast<const UnitInfo *>(st + 2 * L::kKV + L::kQ + L::kScales);
    const int flags = info->flags;
    if (flags & kFirst) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      vref = 0.f;
      coef[0] = coef[1] = p.scale_log2;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        // dims of this lane's part of k-step s: 16-bit pools in order; 8-bit
        // pools 4 neighbouring dims of chunk 4 (s / 4) + c
        const int d0 = Q8 ? (4 * (s / 4) + c) * 16 + 4 * (s % 4) : s * 16 + 2 * c;
        const int d1 = Q8 ? d0 + 2 : d0 + 8;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = r + (k & 1) * 8, d = k & 2 ? d1 : d0;
          const int ch = d >> 3;
          qf[s][k] = lds32(sq + row * D * 2 + (((ch & ~7) | ((ch ^ row) & 7)) << 4) + (d & 7) * 2);
        }
      }
      if (Q8 && std::is_same<T, Bf16>::value) {
        // bf16 -> fp16, each row times the power of two that brings its largest
        // element to [1, 2)
        uint32_t big[2] = {0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < 4; ++k) big[k & 1] = __vmaxu2(big[k & 1], qf[s][k] & 0x7fff7fffu);
        float to[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t b = max(big[h] & 0xffffu, big[h] >> 16);
          b = max(b, __shfl_xor_sync(0xffffffffu, b, 1));
          b = max(b, __shfl_xor_sync(0xffffffffu, b, 2));
          const int e = min(max(static_cast<int>(b >> 7), 1), 253);  // biased exponent
          to[h] = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          coef[h] = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(e) << 23);
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = Bf16::unpack(qf[s][k]);
            qf[s][k] = Fp16::pack(f.x * to[k & 1], f.y * to[k & 1]);
          }
      }
    }

    // scores of this warp's 16 tokens
    const int t0 = warp * 16;
    float sc[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) sc[n][j] = 0.f;
    if (Q8) {
#pragma unroll
      for (int h = 0; h < KS / 4; ++h) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const uint4 w = lds128(sk + chunk_at<D, true>(t0 + 8 * n + r, 4 * h + c));
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) mma16816<false>(sc[n], qf[4 * h + i], e4m3_lo(x[i]), e4m3_hi(x[i]));
        }
      }
    } else {
      const int mi = lane >> 3, row = t0 + (lane & 7) + (mi & 2) * 4;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint32_t b[4];
        ldmatrix4(b, sk + chunk_at<D, false>(row, 2 * s + (mi & 1)));
        mma16816<BF>(sc[0], qf[s], b[0], b[1]);
        mma16816<BF>(sc[1], qf[s], b[2], b[3]);
      }
    }
    const uint32_t valid = (info->valid[t0 >> 5] >> (t0 & 31)) & 0xffffu;
    const int base = info->base + t0;
    bool seen[2][4];
    float vs[2][2];
    float top[2] = {-INFINITY, -INFINITY}, vtop = vref;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float ks[2] = {1.f, 1.f};
      if (Q8) {
        const uint2 a = lds64(ss + (t0 + 8 * n + 2 * c) * 4), b = lds64(ss + kTile * 4 + (t0 + 8 * n + 2 * c) * 4);
        ks[0] = __uint_as_float(a.x);
        ks[1] = __uint_as_float(a.y);
        vs[n][0] = __uint_as_float(b.x);
        vs[n][1] = __uint_as_float(b.y);
        vtop = fmaxf(vtop, fmaxf(vs[n][0], vs[n][1]));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int tok = 8 * n + 2 * c + (j & 1), h = j >> 1;
        seen[n][j] = (valid >> tok) & 1u;
        if (flags & kRagged) {
          const int row = info->row0 + r + 8 * h;
          const int t = p.by_group.div(min(row, info->rows - 1));
          seen[n][j] = seen[n][j] && sees(p, info->pos0 + t, base + tok);
        }
        const float x = sc[n][j] * (Q8 ? coef[h] * ks[j & 1] : coef[h]);
        sc[n][j] = seen[n][j] ? x : -INFINITY;
        top[h] = fmaxf(top[h], sc[n][j]);
      }
    }
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], d));
      top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], d));
      if (Q8) vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, d));
    }
    float keep[2], off[2];
    const float vkeep = Q8 && vref != vtop ? vref / vtop : 1.f;
    const float vinv = Q8 && vtop > 0.f ? 1.f / vtop : 0.f;
    vref = vtop;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float to = fmaxf(m[h], top[h]);
      const float ref = to == -INFINITY ? 0.f : to;  // nothing seen yet: all weights are 2^-inf = 0
      keep[h] = fast_exp2(m[h] - ref);
      off[h] = kLift - ref;
      m[h] = to;
      l[h] *= keep[h];
      keep[h] *= vkeep;
    }
    if (__any_sync(0xffffffffu, keep[0] != 1.f || keep[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        acc[i][0] *= keep[0];
        acc[i][1] *= keep[0];
        acc[i][2] *= keep[1];
        acc[i][3] *= keep[1];
      }
    }
    uint32_t pf[4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        e[j] = fast_exp2(sc[n][j] + off[j >> 1]);
        l[j >> 1] += e[j];
        if (Q8) e[j] *= vs[n][j & 1] * vinv;
      }
      pf[2 * n] = BF ? Bf16::pack(e[0], e[1]) : Fp16::pack(e[0], e[1]);
      pf[2 * n + 1] = BF ? Bf16::pack(e[2], e[3]) : Fp16::pack(e[2], e[3]);
    }

    // weights times values
    uint32_t bad = 0;  // ragged tiles: this lane's tokens (2c, 2c+1, 2c+8, 2c+9) with an infinity or NaN in V
    auto multiply = [&](int j, uint32_t b0, uint32_t b1) {
      if (flags & kRagged) bad |= drop_nonfinite<BF>(b0) | drop_nonfinite<BF>(b1) << 2;
      mma16816<BF>(acc[j], pf, b0, b1);
    };
    if (Q8) {
      constexpr int NV = D >= 128 ? D / 128 : 1;  // 16-byte chunks of V per token and lane
      if (D == 64) {
        uint2 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int tok = t0 + 2 * c + (k & 1) + (k & 2) * 4;
          w[k] = lds64(sv + chunk_at<D, true>(tok, r >> 1) + (r & 1) * 8);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t a = i ? w[0].y : w[0].x, b = i ? w[1].y : w[1].x, e = i ? w[2].y : w[2].x,
                         f = i ? w[3].y : w[3].x;
          const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
          const uint32_t ef0 = __byte_perm(e, f, 0x5140), ef1 = __byte_perm(e, f, 0x7362);
          multiply(4 * i + 0, e4m3_lo(ab0), e4m3_lo(ef0));
          multiply(4 * i + 1, e4m3_hi(ab0), e4m3_hi(ef0));
          multiply(4 * i + 2, e4m3_lo(ab1), e4m3_lo(ef1));
          multiply(4 * i + 3, e4m3_hi(ab1), e4m3_hi(ef1));
        }
      } else {
#pragma unroll
        for (int h = 0; h < NV; ++h) {
          uint32_t w[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int tok = t0 + 2 * c + (k & 1) + (k & 2) * 4;
            const uint4 x = lds128(sv + chunk_at<D, true>(tok, r + 8 * h));
            w[k][0] = x.x;
            w[k][1] = x.y;
            w[k][2] = x.z;
            w[k][3] = x.w;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t ab0 = __byte_perm(w[0][i], w[1][i], 0x5140), ab1 = __byte_perm(w[0][i], w[1][i], 0x7362);
            const uint32_t ef0 = __byte_perm(w[2][i], w[3][i], 0x5140), ef1 = __byte_perm(w[2][i], w[3][i], 0x7362);
            multiply(16 * h + 4 * i + 0, e4m3_lo(ab0), e4m3_lo(ef0));
            multiply(16 * h + 4 * i + 1, e4m3_hi(ab0), e4m3_hi(ef0));
            multiply(16 * h + 4 * i + 2, e4m3_lo(ab1), e4m3_lo(ef1));
            multiply(16 * h + 4 * i + 3, e4m3_hi(ab1), e4m3_hi(ef1));
          }
        }
      }
    } else {
      const int mi = lane >> 3, row = t0 + (lane & 7) + (mi & 1) * 8;
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        uint32_t b[4];
        ldmatrix4_trans(b, sv + chunk_at<D, false>(row, j + (mi >> 1)));
        multiply(j, b[0], b[1]);
        multiply(j + 1, b[2], b[3]);
      }
    }
    if (flags & kRagged) {
      // bits of the lanes that hold the same tokens' other dims
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) bad |= __shfl_xor_sync(0xffffffffu, bad, d);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (seen[n][j] && (bad >> (2 * n + (j & 1)) & 1u)) l[j >> 1] = NAN;
    }

    const bool last = flags & kLast;
    const int head = info->head, row0 = info->row0, rows = info->rows, part = info->part;
    const int64_t q0 = info->q0;
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + stage);
    if (++stage == L::kStages) {
      stage = 0;
      phase ^= 1;
    }
    if (!last) continue;

    // Join the four warps: 2 and 3 into 0 and 1, then 1 into 0.
#pragma unroll
    for (int d = 1; d < 4; d <<= 1) {
      l[0] += __shfl_xor_sync(0xffffffffu, l[0], d);
      l[1] += __shfl_xor_sync(0xffffffffu, l[1], d);
    }
    if (Q8) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] *= vref;
    }
    float *stats = merge + 2 * kRows * D;  // [2][2][16]: maximum and sum of a giving warp's rows
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(joined);
      const bool ok = mbar_wait_bounded(joined, join_phase, kBulkWaitLimitNs);
      join_phase ^= 1;
      if (!ok && lane == 0) raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
      return ok;
    };
    auto give = [&](int to) {
      float *a = merge + to * kRows * D, *b = stats + to * 2 * kRows;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) a[(i * 4 + j) * 32 + lane] = acc[i][j];
      if (c == 0) {
        b[r] = m[0];
        b[r + 8] = m[1];
        b[kRows + r] = l[0];
        b[kRows + r + 8] = l[1];
      }
    };
    auto take = [&](int from) {
      const float *a = merge + from * kRows * D, *b = stats + from * 2 * kRows;
      float mine[2], theirs[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float om = b[r + 8 * h], to = fmaxf(m[h], om), ref = to == -INFINITY ? 0.f : to;
        mine[h] = fast_exp2(m[h] - ref);
        theirs[h] = fast_exp2(om - ref);
        m[h] = to;
        l[h] = l[h] * mine[h] + b[kRows + r + 8 * h] * theirs[h];
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = acc[i][j] * mine[j >> 1] + a[(i * 4 + j) * 32 + lane] * theirs[j >> 1];
    };
    if (warp >= 2) give(warp - 2);
    if (!meet()) return;
    if (warp < 2) take(warp);
    if (!meet()) return;
    if (warp == 1) give(0);
    if (!meet()) return;
    if (warp == 0) take(0);
    if (!meet()) return;  // before the next give
    if (warp == 0) {
      if (flags & kWhole) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = row0 + r + 8 * h;
          const int t = p.by_group.div(row), g = row - t * p.group;
          if (row >= rows || q0 + t >= p.num_tokens) continue;
          char *out = p.o + (q0 + t) * p.o_row_stride + (static_cast<int64_t>(head) * p.group + g) * p.o_head_stride;
          const float inv = l[h] == 0.f ? 0.f : 1.f / l[h];
          if (Q8) {
            // lane c of a row holds dims (2c + k) W .. + W of each W * 8 dims, W neighbouring n-tiles
            constexpr int W = D >= 128 ? 16 : 8;
#pragma unroll
            for (int b = 0; b < NT / W; ++b)
#pragma unroll
              for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int i = 0; i < W; i += 8) {
                  uint32_t w[4];
#pragma unroll
                  for (int x = 0; x < 4; ++x)
                    w[x] = T::pack(acc[b * W + i + 2 * x][2 * h + k] * inv, acc[b * W + i + 2 * x + 1][2 * h + k] * inv);
                  *reinterpret_cast<uint4 *>(out + (b * W * 8 + (2 * c + k) * W + i) * 2) =
                      make_uint4(w[0], w[1], w[2], w[3]);
                }
          } else {
#pragma unroll
            for (int i = 0; i < NT; ++i)
              *reinterpret_cast<uint32_t *>(out + (i * 8 + 2 * c) * 2) =
                  T::pack(acc[i][2 * h] * inv, acc[i][2 * h + 1] * inv);
          }
        }
      } else {
        // in the order of the registers: the joining kernel knows it
        float *a = p.partials + static_cast<int64_t>(part) * (kRows * D + 2 * kRows), *b = a + kRows * D;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = r + 8 * h;
          if (row0 + row >= rows) continue;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            float2 *at;
            float x, y;
            if (Q8) {
              constexpr int W = D >= 128 ? 16 : 8;
              // pairs of neighbouring n-tiles are neighbouring dims
              const int k = i & 1, j = i & ~1;
              at = reinterpret_cast<float2 *>(a + row * D + (j / W) * W * 8 + (2 * c + k) * W + j % W);
              x = acc[j][2 * h + k];
              y = acc[j + 1][2 * h + k];
            } else {
              at = reinterpret_cast<float2 *>(a + row * D + i * 8 + 2 * c);
              x = acc[i][2 * h];
              y = acc[i][2 * h + 1];
            }
            *at = make_float2(x, y);
          }
          if (c == 0) {
            b[row] = m[h];
            b[kRows + row] = l[h];
          }
        }
      }
    }
  }
}

template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(kThreads, Layout<D, Q8>::kCtas) decode_kernel(const __grid_constant__ AttnParams p) {
  using L = Layout<D, Q8>;
  extern __shared__ uint8_t raw[];
  uint8_t *smem = raw + ((128 - (smem_addr(raw) & 127)) & 127);
  uint8_t *stages = smem;
  float *merge = reinterpret_cast<float *>(smem + L::kStages * L::kStage);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kStages * L::kStage + L::kMerge + 256);
  uint64_t *empty = full + L::kStages, *joined = empty + L::kStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(full + i, 33);  // the loading warp's copies, and its descriptor
      mbar_init(empty + i, kConsumers);
    }
    mbar_init(joined, kConsumers);
  }
  pdl_wait();
  Place place;
  const bool work = find_place(p, place);  // synchronises the block
  pdl_trigger();
  if (!work) {
    if (threadIdx.x == 0) p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  if (threadIdx.x >= kConsumers * 32)
    load_units<D, Q8>(p, place, stages, full, empty);
  else
    compute_units<T, D, Q8>(p, place, stages, full, empty, joined, merge);
}

// Joins the parts of a result that began in CTA c - 1 and goes on in CTA c (and
// maybe further): part 2 (c - 1) + 1, then the first parts of the CTAs that
// follow.  One block per (c, query row); 32 lanes per part, parts in turn over
// the warps, then the warps in order.
constexpr int kJoinWarps = 4;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ AttnParams p) {
  constexpr int N = D / 32;
  __shared__ float part[kJoinWarps][D + 2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x + 1, r = blockIdx.y;
  pdl_wait();
  const int4 meta = p.meta[c];
  const int n = meta.x, row = (meta.z & 0xffff) + r, head = meta.z >> 16;
  if (n == 0 || row >= meta.w) return;
  const int64_t stride = kRows * D + 2 * kRows;
  const float *base = p.partials + static_cast<int64_t>(2 * (c - 1)) * stride;
  auto at = [&](int k) { return base + (k == 0 ? 1 : 2 * k) * stride; };
  float m = -INFINITY;
  for (int k = lane; k < n; k += 32) m = fmaxf(m, at(k)[kRows * D + r]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  const float ref = m == -INFINITY ? 0.f : m;
  float acc[N], l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int k = warp; k < n; k += kJoinWarps) {
    const float *a = at(k);
    const float w = fast_exp2(a[kRows * D + r] - ref);
    l += a[kRows * D + kRows + r] * w;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 x = *reinterpret_cast<const float2 *>(a + r * D + i * 32 + 2 * lane);
      acc[i] += x.x * w;
      acc[i + 1] += x.y * w;
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) part[warp][i * 32 + lane] = acc[i];
  if (lane == 0) part[warp][D] = l;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) {
    l += part[w][D];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += part[w][i * 32 + lane];
  }
  const int t = p.by_group.div(row), g = row - t * p.group;
  if (meta.y + static_cast<int64_t>(t) >= p.num_tokens) return;
  char *out = p.o + (meta.y + static_cast<int64_t>(t)) * p.o_row_stride +
              (static_cast<int64_t>(head) * p.group + g) * p.o_head_stride;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < N; i += 2)
    *reinterpret_cast<uint32_t *>(out + (i * 32 + 2 * lane) * 2) = T::pack(acc[i] * inv, acc[i + 1] * inv);
}

// The grid of the decode kernel and the bytes of its parts.
int decode_ctas(int D, bool q8) {
  int per_sm = 1;
  if (D == 64) per_sm = q8 ? Layout<64, true>::kCtas : Layout<64, false>::kCtas;
  if (D == 128) per_sm = q8 ? Layout<128, true>::kCtas : Layout<128, false>::kCtas;
  if (D == 256) per_sm = q8 ? Layout<256, true>::kCtas : Layout<256, false>::kCtas;
  return sm_count() * per_sm;
}

// Shared memory above 48 KB is asked for once per kernel and device.
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

template <typename T, int D, bool Q8>
int launch(AttnParams &p, int ctas, int rows, cudaStream_t stream) {
  int rc = allow_smem(reinterpret_cast<const void *>(decode_kernel<T, D, Q8>), Layout<D, Q8>::kSmem);
  if (rc != YL_OK) return rc;
  rc = launch_dependent(decode_kernel<T, D, Q8>, dim3(ctas), dim3(kThreads), Layout<D, Q8>::kSmem, stream,
                        "yl_paged_attention launch", p);
  if (rc != YL_OK) return rc;
  return launch_dependent(join_kernel<T, D>, dim3(ctas - 1, rows), dim3(kJoinWarps * 32), 0,
                          stream, "yl_paged_attention launch", p);
}

}  // namespace

int64_t decode_workspace(const yl_paged_attention_args *a) {
  const int64_t ctas = decode_ctas(a->head_dim, a->kv_dtype == YL_KV_E4M3);
  return ctas * 16 + ctas * 2 * (kRows * a->head_dim + 2 * kRows) * 4;
}

int launch_decode(AttnParams &p, const yl_paged_attention_args *a, int64_t most_rows, cudaStream_t stream) {
  const bool q8 = a->kv_dtype == YL_KV_E4M3;
  const int ctas = decode_ctas(a->head_dim, q8);
  const int rows = static_cast<int>(std::min<int64_t>(most_rows, kRows));
  p.meta = static_cast<int4 *>(a->workspace);
  p.partials = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + ctas * 16);
  auto go = [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    return q8 ? launch<T, D, true>(p, ctas, rows, stream) : launch<T, D, false>(p, ctas, rows, stream);
  };
  auto dim = [&](auto t) {
    if (a->head_dim == 64) return go(t, std::integral_constant<int, 64>{});
    if (a->head_dim == 128) return go(t, std::integral_constant<int, 128>{});
    return go(t, std::integral_constant<int, 256>{});
  };
  return a->dtype == YL_DTYPE_BF16 ? dim(Bf16{}) : dim(Fp16{});
}

}  // namespace ylk
