// Paged attention of sequences with few new tokens (decode), for sm_100a.
//
// The keys and values are read once and the arithmetic is small, so HBM bounds
// it: 2 * visible tokens * head_dim * item bytes per KV head.  What the design
// is for is keeping every SM's loads in flight to the end:
//
// * The batch's work is one line of units, a unit being a tile of visible tokens
//   (128 where a head's row is 128 bytes or less, else 64) of one (sequence, KV
//   head, 8 or 16 query rows); the query rows of a unit are the new tokens times
//   the heads of the group.  Each CTA takes an equal run of that line, whatever
//   the lengths of the sequences; each finds its place by scanning the batch
//   itself (a few KB), so a call needs no plan.
//   A (sequence, head) whose units fall in several CTAs leaves its parts in the
//   workspace, and a second kernel joins them, in a fixed order.
// * Four warps of a CTA only issue loads, a quarter of a unit's tokens each: they
//   walk the units, look up pages one unit ahead, and fill a ring of stages with
//   16-byte asynchronous copies, across the ends of sequences.  (One such warp
//   spent 3,300 cycles on a unit whose bytes HBM delivers in 1,500.)  Tokens that
//   no query sees are zero-filled, not read.
// * Four warps compute, each on its own quarter of the tile with its own
//   reference, sum and accumulator (online softmax); the four are joined when a
//   (sequence, head) ends.  The reference is the running maximum, but moves only
//   when some score of the step passes it by 2^4 or more: the common step has one
//   vote instead of nine shuffles, two exponentials of the factor and a division
//   (357 -> 346 us for 256 sequences of 8-bit pages).  Products are m16n8k16
//   matrix instructions with the 16 rows along the tokens (k.q) or the head
//   dimension (v.p) and 8 columns of query rows: at 1 to 16 query rows this
//   wastes least, where a 128-row tensor tile would be padding.  The weights turn
//   from the first product's result to the second's operand by a transposing
//   register move.
// * An 8-bit pool is multiplied in fp16: every e4m3 value is exact there.  bf16
//   queries are first brought into fp16's range by a power of two per row, exact
//   for all elements within 2^-17 of the row's largest (8 bits above fp16's
//   smallest step) and off by up to 2^-25 of it below.  The contraction order of
//   k.q is free, so a lane takes 4 neighbouring codes as its part of a k-step and
//   K needs no transposition; the codes of two tokens of V are interleaved by byte
//   permutes before conversion.  K's scale multiplies the scores; V's scale,
//   relative to the largest seen so far, multiplies the weights before they are
//   rounded.  Weights are kept times 2^11, so the largest is at most 2^15, and
//   times V's scale their smallest steps are 2^-35 of the largest weight times the
//   largest scale.
// * All sums, maxima and accumulators are fp32; weights are rounded once, to
//   fp16 (8-bit and fp16 pools) or bf16 (bf16 pools), as the matrix
//   instructions take them.
//
// Measured, 256 sequences of 128 to 8k tokens, 8 KV heads of 128: 8-bit pages
// 379 us in a loop of seconds, where the power limit lowers the clock, 5.5 TB/s of
// 6.46 that a plain copy reaches; in a burst 340, 6.1 TB/s; the loads alone take
// 313, the arithmetic alone 334 before its last step.  16-bit pages 627 us, 6.6
// TB/s; head_dim 256 660 us, 6.3 TB/s; head_dim 64 252 us, 4.1 TB/s, where the
// softmax of a score costs as much as at 128 and carries half the bytes.  Pages
// of one token 566 us: an id, an address and a scale each in the loading warps.
// One sequence of 8k tokens takes 13 us: two launches and one chain of loads.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "attend_device.cuh"
#include "tma.cuh"

namespace ylk {
namespace {

constexpr int kConsumers = 4;  // warps that compute, a quarter of a unit's tokens each
constexpr int kThreads = 2 * kConsumers * 32;  // and as many that load
// A CTA's run is at least this many units, so that a short sequence is not cut
// into parts whose joining costs more than they save.
constexpr int kMinRun = 2;

// Unit descriptor in a stage, written by the loading warps.
struct UnitInfo {
  uint32_t valid[4];  // of a quarter of the tile: tokens that some query sees, with a good page
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

// NB: blocks of 8 query rows of a unit.
template <int D, bool Q8, int NB>
struct Layout {
  static constexpr int kItem = Q8 ? 1 : 2;
  static constexpr int kRow = D * kItem;            // bytes of a token's head row
  static constexpr int kChunks = kRow / 16;         // 16-byte chunks of it
  static constexpr int kTokens = kRow <= 128 ? 32 : 16;  // of a computing warp: 8 KB of K and V or less, but for kRow 512
  static constexpr int kTile = kConsumers * kTokens;
  static constexpr int kRows = 8 * NB;              // query rows of a unit
  static constexpr int kKV = kTile * kRow;          // bytes of K (or V) in a stage
  static constexpr int kQ = kRows * D * 2;
  static constexpr int kScales = Q8 ? 2 * kTile * 4 : 0;
  static constexpr int kInfo = 2 * kKV + kQ + kScales;
  static constexpr int kStage = kInfo + 128;
  static constexpr int kMerge = 2 * (kRows * D + 2 * kRows) * 4;  // two warps' accumulators, maxima and sums
  static constexpr int kRest = 128 + 256;           // alignment of the stages, barriers
  // two CTAs per SM where two stages and more fit each
  static constexpr int kCtas = kStage * 2 + kMerge + kRest <= 113 * 1024 ? 2 : 1;
  static constexpr int kBudget = (kCtas == 2 ? 113 : 226) * 1024 - kMerge - kRest;
  static constexpr int kStages = kBudget / kStage > 8 ? 8 : kBudget / kStage;
  static constexpr int kSmem = kStages * kStage + kMerge + kRest;
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
  return r * (D * (Q8 ? 1 : 2)) + (((c & ~7) | ((c ^ f) & 7)) << 4);
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

// An 8 x 8 matrix of 16-bit values turned over, in the layout of a fragment.
__device__ __forceinline__ uint32_t turn(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Zero what is no finite number in the V rows [t0, t0 + TOKENS) of a tile, so
// that weight 0 times it is 0; returns which of the tokens had any.  Only for
// tiles of which some query does not see all: elsewhere it belongs in the
// result.
template <int D, bool Q8, bool BF, int TOKENS>
__device__ __noinline__ uint32_t clean_values(uint32_t sv, int t0) {
  constexpr uint32_t inf = BF ? 0x7f807f80u : 0x7c007c00u;
  constexpr int kChunks = D * (Q8 ? 1 : 2) / 16;
  const int lane = threadIdx.x & 31;
  uint32_t bad = 0;
#pragma unroll 1
  for (int n = lane; n < TOKENS * kChunks; n += 32) {
    const int t = n % TOKENS;
    const uint32_t at = sv + chunk_at<D, Q8>(t0 + t, n / TOKENS);
    uint4 w = lds128(at);
    uint32_t any = 0;
    auto clean = [&](uint32_t &x) {
      const uint32_t mask = Q8 ? __vcmpeq4(x & 0x7f7f7f7fu, 0x7f7f7f7fu) : __vcmpgeu2(x & 0x7fff7fffu, inf);
      any |= mask;
      x &= ~mask;
    };
    clean(w.x);
    clean(w.y);
    clean(w.z);
    clean(w.w);
    if (any) {
      bad |= 1u << t;
      asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
    }
  }
  bad = __reduce_or_sync(0xffffffffu, bad);
  __syncwarp();
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

template <class L>
__device__ __forceinline__ SeqWork work_of(const AttnParams &p, const Seq &s) {
  constexpr int kRows = L::kRows, kTile = L::kTile;
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
template <class L>
__device__ __forceinline__ bool find_place(const AttnParams &p, Place &out) {
  __shared__ int64_t warp_sum[kThreads / 32];
  __shared__ Place found;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int m = (p.batch + kThreads - 1) / kThreads;
  const int lo = min(tid * m, p.batch), hi = min(lo + m, p.batch);
  int64_t sum = 0;
  for (int i = lo; i < hi; ++i) sum += work_of<L>(p, load_seq(p, i, blockIdx.x == 0)).units;
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
      const int64_t u = work_of<L>(p, load_seq(p, i, false)).units;
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
// Loading warps
// ---------------------------------------------------------------------------
template <int D, bool Q8, int NB>
__device__ __forceinline__ void load_units(const AttnParams &p, const Place &place, uint8_t *stages, uint64_t *full,
                                           uint64_t *empty) {
  using L = Layout<D, Q8, NB>;
  constexpr int kTile = L::kTile, kRows = L::kRows, kTokens = L::kTokens;  // kTokens at most one per lane
  const int lane = threadIdx.x & 31, quarter = (threadIdx.x >> 5) - kConsumers;
  const int my = quarter * kTokens + lane;  // this lane's token of a tile
  const int64_t first = place.run * blockIdx.x;
  const int count = static_cast<int>(min(place.run, place.total - first));
  int i = place.seq;
  Seq s = load_seq(p, i, false);
  SeqWork w = work_of<L>(p, s);
  int64_t begin = place.start;  // units before sequence i
  int tile = static_cast<int>(place.within % w.tiles);
  int64_t rest = place.within / w.tiles;
  int rt = static_cast<int>(rest % w.row_tiles);
  int head = static_cast<int>(rest / w.row_tiles);
  Span v = span_of(p, s, 0, s.fresh);

  // the page id of the lane's token, looked up one unit ahead
  constexpr int kUnused = -0x7fffffff, kNoEntry = -0x7ffffffe;  // not a token of the tile; no such entry
  int base, cnt, page, ord;
  auto look_up = [&]() {
    const bool in_head = tile < w.head_tiles;
    base = (in_head ? 0 : v.low) + (in_head ? tile : tile - w.head_tiles) * kTile;
    cnt = min(kTile, (in_head ? v.head : v.end) - base);
    page = kUnused;
    if (lane < kTokens && my < cnt) {
      ord = p.by_page.div(base + my);
      const int64_t e = static_cast<int64_t>(s.e0) + ord;
      // (the id is not looked at here, so that the load stays in flight)
      page = e >= 0 && e < p.indices_cap ? __ldg(p.kv_indices + e) : kNoEntry;
    }
  };
  look_up();
  uint32_t phase = 1;  // a fresh stage counts as consumed
  int stage = 0;
  for (int u = 0; u < count; ++u) {
    uint8_t *st = stages + stage * L::kStage;
    const uint32_t sk = smem_addr(st), sv = sk + L::kKV, sq = sv + L::kKV, ss = sq + L::kQ;
    UnitInfo *info = reinterpret_cast<UnitInfo *>(st + L::kInfo);
    const bool ok = page >= 0 && page < p.num_pages;
    if (!ok && page != kUnused)
      raise_deverr(p.error_word, page == kNoEntry ? YL_DEVERR_INDICES_CAP : YL_DEVERR_PAGE_RANGE);
    const int64_t off = ok ? page * p.page_stride + (base + my - ord * p.page_size) * p.slot_stride + head * p.head_stride : 0;
    const int64_t sc = ok ? page * p.scale_page_stride + head * p.scale_head_stride : 0;
    const uint32_t valid = __ballot_sync(0xffffffffu, ok);
    // this unit's description, before the state moves on
    const bool is_first = u == 0 || tile == 0, ends = tile == w.tiles - 1;
    const int rows = s.fresh * p.group, row0 = rt * kRows, pos0 = s.first, q0 = s.q0, u_base = base, u_head = head;
    const int64_t seg = begin + (static_cast<int64_t>(head) * w.row_tiles + rt) * w.tiles;  // its first unit in the line
    int flags = is_first ? kFirst : 0;
    if (ends || u == count - 1) flags |= kLast;
    if (ends && seg >= first) flags |= kWhole;
    const int last_pos = max(s.first + s.fresh - 1, -1), end = base + cnt - 1;
    const bool all = end <= pos0 && (p.window == 0 || base > last_pos - p.window || end < p.sinks);
    if (s.fresh > 1 && !all) flags |= kRagged;
    if (u == 0 && quarter == 0 && lane == 0) {
      // where the parts of a result lie that began in an earlier CTA
      int4 meta = make_int4(0, 0, 0, 0);
      if (seg < first) {
        const int c0 = static_cast<int>(seg / place.run), c1 = static_cast<int>((seg + w.tiles - 1) / place.run);
        // the first CTA boundary inside it stands for the whole of it
        if (c0 + 1 == static_cast<int>(blockIdx.x)) meta = make_int4(c1 - c0 + 1, q0, row0 | head << 16, rows);
      }
      p.meta[blockIdx.x] = meta;
    }
    // on to the next unit's look-up, in flight while this one is copied
    if (u + 1 < count) {
      if (++tile == w.tiles) {
        tile = 0;
        if (++rt == w.row_tiles) {
          rt = 0;
          if (++head == p.heads) {
            head = 0;
            begin += w.units;
            do {  // ends: count units remain in the line
              s = load_seq(p, ++i, false);
              w = work_of<L>(p, s);
            } while (w.units == 0 && i + 1 < p.batch);
            v = span_of(p, s, 0, s.fresh);
          }
        }
      }
      look_up();
    }
    if (!mbar_wait_clocked(empty + stage, phase)) {
      if (lane == 0) raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
      break;
    }
    constexpr int kRowsPer = 32 / L::kChunks;  // rows of one copy instruction
    const int c = lane % L::kChunks;
    const bool whole = valid == (kTokens == 32 ? 0xffffffffu : 0xffffu);
    if (whole && (p.page_size & 15) == 0 && ((u_base + quarter * kTokens) & 15) == 0) {
      // pages of a multiple of 16 tokens: 16 rows lie a constant stride apart,
      // one address each 16 rows instead of one a row
      const int64_t mine = (lane / L::kChunks) * p.slot_stride + c * 16, other = p.kv[1] - p.kv[0];
#pragma unroll
      for (int g = 0; g < kTokens / 16; ++g) {
        const char *src = p.kv[0] + __shfl_sync(0xffffffffu, off, 16 * g) + mine;
#pragma unroll
        for (int j = 0; j < 16 / kRowsPer; ++j) {
          const int at = chunk_at<D, Q8>(quarter * kTokens + 16 * g + j * kRowsPer + lane / L::kChunks, c);
          cp_async16(sk + at, src, true);
          cp_async16(sv + at, src + other, true);
          src += kRowsPer * p.slot_stride;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < kTokens / kRowsPer; ++j) {
        const int r = j * kRowsPer + lane / L::kChunks;
        const int64_t o = __shfl_sync(0xffffffffu, off, r) + c * 16;
        const bool good = (valid >> r) & 1u;
        const int at = chunk_at<D, Q8>(quarter * kTokens + r, c);
        cp_async16(sk + at, p.kv[0] + o, good);
        cp_async16(sv + at, p.kv[1] + o, good);
      }
    }
    if (Q8 && lane < kTokens) {
      cp_async4(ss + my * 4, p.scale[0] + sc, ok);
      cp_async4(ss + (kTile + my) * 4, p.scale[1] + sc, ok);
    }
    if (is_first) {
      constexpr int kQChunks = D / 8;
#pragma unroll
      for (int j = 0; j < (kRows * kQChunks + 127) / 128; ++j) {
        const int n = (j * kConsumers + quarter) * 32 + lane, r = n / kQChunks, qc = n % kQChunks;
        if (n >= kRows * kQChunks) break;
        const int row = row0 + r;
        const int t = p.by_group.div(row), g = row - t * p.group;
        const int64_t qrow = static_cast<int64_t>(q0) + t;
        const bool has = row < rows && qrow < p.num_tokens;
        const char *src =
            p.q + (has ? qrow * p.q_row_stride + (static_cast<int64_t>(u_head) * p.group + g) * p.q_head_stride : 0) + qc * 16;
        cp_async16(sq + r * D * 2 + (((qc & ~7) | ((qc ^ r) & 7)) << 4), src, has);
      }
    }
    cp_async_arrive(smem_addr(full + stage));
    if (lane == 0) {
      info->valid[quarter] = valid;
      if (quarter == 0) {
        info->base = u_base;
        info->pos0 = pos0;
        info->row0 = row0;
        info->rows = rows;
        info->q0 = q0;
        info->head = u_head;
        info->flags = flags;
        info->part = static_cast<int>(2 * blockIdx.x + (seg >= first ? 1 : 0));
      }
      mbar_arrive(full + stage);
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
template <typename T, int D, bool Q8, int NB>
__device__ __forceinline__ void compute_units(const AttnParams &p, const Place &place, uint8_t *stages, uint64_t *full,
                                              uint64_t *empty, uint64_t *joined, float *merge) {
  using L = Layout<D, Q8, NB>;
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;  // type of the matrix instructions
  constexpr int KS = D / 16;                                // k-steps of k.q
  constexpr int MT = L::kTokens / 16;                       // token tiles of this warp
  constexpr int DT = D / 16;                                // tiles of the head dimension
  constexpr int W = D >= 128 ? 16 : 8;                      // codes of V that a lane takes at once
  constexpr int kTile = L::kTile, kRows = L::kRows;
  // Weights are kept times 2^kLift; a score may pass its row's reference by
  // kSlack (as log2) before the reference moves.  2^(11 + 4) is in fp16's range.
  constexpr float kLift = BF ? 0.f : 11.f, kSlack = 4.f;
  constexpr float kUnset = 3.0e38f;  // `off` of a row that has seen nothing: every score passes it
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int t0 = warp * L::kTokens;
  const int64_t first = place.run * blockIdx.x;
  const int count = static_cast<int>(min(place.run, place.total - first));
  uint32_t qf[KS][NB][2];
  // columns of a fragment: query rows 8 b + 2 c and 8 b + 2 c + 1
  // m: a row's reference, off = kLift - m; vref, vinv: V's reference scale, one over it
  float acc[DT][NB][4], m[NB][2], off[NB][2], l[NB][2], coef[NB][2], vref = 0.f, vinv = 0.f;
  int stage = 0;
  uint32_t phase = 0, join_phase = 0;
  for (int u = 0; u < count; ++u) {
    uint8_t *st = stages + stage * L::kStage;
    const uint32_t sk = smem_addr(st), sv = sk + L::kKV, sq = sv + L::kKV, ss = sq + L::kQ;
    if (!mbar_wait_clocked(full + stage, phase)) {
      if (lane == 0) raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
      return;
    }
    const UnitInfo *info = reinterpret_cast<const UnitInfo *>(st + L::kInfo);
    const int flags = info->flags;
    if (flags & kFirst) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][b][j] = 0.f;
        m[b][0] = m[b][1] = -INFINITY;
        off[b][0] = off[b][1] = kUnset;
        l[b][0] = l[b][1] = 0.f;
        coef[b][0] = coef[b][1] = p.scale_log2;
        const int row = 8 * b + r;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          // dims of this lane's part of k-step s: 16-bit pools in order; 8-bit
          // pools 4 neighbouring dims of chunk 4 (s / 4) + c
          const int d0 = Q8 ? (4 * (s / 4) + c) * 16 + 4 * (s % 4) : s * 16 + 2 * c;
          const int d1 = Q8 ? d0 + 2 : d0 + 8;
          auto at = [&](int d) { return sq + row * D * 2 + ((((d >> 3) & ~7) | (((d >> 3) ^ row) & 7)) << 4) + (d & 7) * 2; };
          qf[s][b][0] = lds32(at(d0));
          qf[s][b][1] = lds32(at(d1));
        }
        if (Q8 && std::is_same<T, Bf16>::value) {
          // bf16 -> fp16, each row times the power of two that brings its
          // largest element to [1, 2)
          uint32_t big = 0;
#pragma unroll
          for (int s = 0; s < KS; ++s) big = __vmaxu2(big, __vmaxu2(qf[s][b][0] & 0x7fff7fffu, qf[s][b][1] & 0x7fff7fffu));
          big = max(big & 0xffffu, big >> 16);
          big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
          big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
          const int e = min(max(static_cast<int>(big >> 7), 1), 253);  // biased exponent
          const float to = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
          const float back = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(e) << 23);
          coef[b][0] = __shfl_sync(0xffffffffu, back, 8 * c);
          coef[b][1] = __shfl_sync(0xffffffffu, back, 8 * c + 4);
#pragma unroll
          for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float2 f = Bf16::unpack(qf[s][b][k]);
              qf[s][b][k] = Fp16::pack(f.x * to, f.y * to);
            }
        }
      }
      vref = vinv = 0.f;
    }

    // scores of this warp's tokens
    float sc[MT][NB][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[t][b][j] = 0.f;
    if (Q8) {
#pragma unroll
      for (int h = 0; h < KS / 4; ++h) {
        uint4 x[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          x[t][0] = lds128(sk + chunk_at<D, true>(t0 + 16 * t + r, 4 * h + c));
          x[t][1] = lds128(sk + chunk_at<D, true>(t0 + 16 * t + r + 8, 4 * h + c));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            const uint32_t w0 = i == 0 ? x[t][0].x : i == 1 ? x[t][0].y : i == 2 ? x[t][0].z : x[t][0].w;
            const uint32_t w1 = i == 0 ? x[t][1].x : i == 1 ? x[t][1].y : i == 2 ? x[t][1].z : x[t][1].w;
            const uint32_t a[4] = {e4m3_lo(w0), e4m3_lo(w1), e4m3_hi(w0), e4m3_hi(w1)};
#pragma unroll
            for (int b = 0; b < NB; ++b) mma16816<false>(sc[t][b], a, qf[4 * h + i][b][0], qf[4 * h + i][b][1]);
          }
      }
    } else {
      const int mi = lane >> 3, row = t0 + (lane & 7) + (mi & 1) * 8;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          uint32_t a[4];
          ldmatrix4(a, sk + chunk_at<D, false>(row + 16 * t, 2 * s + (mi >> 1)));
#pragma unroll
          for (int b = 0; b < NB; ++b) mma16816<BF>(sc[t][b], a, qf[s][b][0], qf[s][b][1]);
        }
    }
    // bit i: token t0 + i of the tile
    const uint32_t valid = info->valid[warp];
    float ks[MT][2], vs[MT][2], x[MT][NB][4];  // x: scores as log2, relative to the reference, lifted
    bool moves = false;
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int tok = t0 + 16 * t + r + 8 * k;
        ks[t][k] = Q8 ? __uint_as_float(lds32(ss + tok * 4)) : 1.f;
        vs[t][k] = Q8 ? __uint_as_float(lds32(ss + (kTile + tok) * 4)) : 1.f;
        if (Q8) moves |= vs[t][k] > vref;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            x[t][b][2 * k + j] = fmaf(sc[t][b][2 * k + j], Q8 ? coef[b][j] * ks[t][k] : coef[b][j], off[b][j]);
      }
    uint32_t ghosts = 0;  // tokens whose V had an infinity or NaN, zeroed in the stage
    if (valid != (L::kTokens == 32 ? 0xffffffffu : 0xffffu)) {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!((valid >> (16 * t + r + 4 * (j & 2))) & 1u)) x[t][b][j] = -INFINITY;
    }
    if (flags & kRagged) {
      ghosts = clean_values<D, Q8, BF, L::kTokens>(sv, t0);
      if (Q8) {  // a V scale that is no number counts like such values
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            if (!is_number(vs[t][k])) {
              vs[t][k] = 0.f;
              ghosts |= 1u << (16 * t + r + 8 * k);
            }
      }
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int pos = info->pos0 + static_cast<int>(p.by_group.div(min(info->row0 + 8 * b + 2 * c + j, info->rows - 1)));
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int tok = 16 * t + r + 8 * k;
              if (!sees(p, pos, info->base + t0 + tok))
                x[t][b][2 * k + j] = -INFINITY;
              else if ((ghosts >> tok) & 1u)
                x[t][b][2 * k + j] = NAN;
            }
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 4; ++j) moves |= x[t][b][j] > kLift + kSlack;
    if (__any_sync(0xffffffffu, moves)) {
      // some row's reference, or V's, moves: to the largest so far
      float vtop = vref;
      if (Q8) {
#pragma unroll
        for (int t = 0; t < MT; ++t) vtop = fmaxf(vtop, fmaxf(vs[t][0], vs[t][1]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, d));
      }
      const float vkeep = Q8 && vref != vtop ? vref / vtop : 1.f;
      vinv = Q8 && vtop > 0.f ? 1.f / vtop : 0.f;
      vref = vtop;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float s[MT][2], top = m[b][j];  // the scores themselves, what is masked left out
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float at = x[t][b][2 * k + j];
              s[t][k] = at > -INFINITY ? sc[t][b][2 * k + j] * (Q8 ? coef[b][j] * ks[t][k] : coef[b][j]) : at;
              top = fmaxf(top, s[t][k]);
            }
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          const float keep = top == -INFINITY ? 1.f : fast_exp2(m[b][j] - top);
          m[b][j] = top;
          off[b][j] = top == -INFINITY ? kUnset : kLift - top;
          l[b][j] *= keep;
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int k = 0; k < 2; ++k) x[t][b][2 * k + j] = s[t][k] + off[b][j];
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            acc[i][b][j] *= keep * vkeep;
            acc[i][b][2 + j] *= keep * vkeep;
          }
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          sc[t][b][j] = fast_exp2(x[t][b][j]);
          sc[t][b][2 + j] = fast_exp2(x[t][b][2 + j]);
          l[b][j] += sc[t][b][j] + sc[t][b][2 + j];
        }
    uint32_t pf[MT][NB][2];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float w = Q8 ? vs[t][k] * vinv : 1.f;
          const float x = sc[t][b][2 * k] * w, y = sc[t][b][2 * k + 1] * w;
          pf[t][b][k] = turn(BF ? Bf16::pack(x, y) : Fp16::pack(x, y));
        }

    // values times weights
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      if (Q8) {
#pragma unroll
        for (int h = 0; h < (D == 256 ? 2 : 1); ++h) {
          uint32_t w[4][W / 4];  // codes of tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int tok = t0 + 16 * t + 2 * c + (k & 1) + (k & 2) * 4;
            if (W == 16) {
              const uint4 x = lds128(sv + chunk_at<D, true>(tok, r + 8 * h));
              w[k][0] = x.x;
              w[k][1] = x.y;
              w[k][W / 4 - 2] = x.z;
              w[k][W / 4 - 1] = x.w;
            } else {
              const uint2 x = lds64(sv + chunk_at<D, true>(tok, r >> 1) + (r & 1) * 8);
              w[k][0] = x.x;
              w[k][1] = x.y;
            }
          }
#pragma unroll
          for (int g = 0; g < W / 4; ++g)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t lo = __byte_perm(w[0][g], w[1][g], i ? 0x7362 : 0x5140);
              const uint32_t hi = __byte_perm(w[2][g], w[3][g], i ? 0x7362 : 0x5140);
              const uint32_t a[4] = {e4m3_lo(lo), e4m3_hi(lo), e4m3_lo(hi), e4m3_hi(hi)};
#pragma unroll
              for (int b = 0; b < NB; ++b) mma16816<false>(acc[8 * h + 2 * g + i][b], a, pf[t][b][0], pf[t][b][1]);
            }
        }
      } else {
        const int mi = lane >> 3, row = t0 + 16 * t + (lane & 7) + (mi >> 1) * 8;
#pragma unroll
        for (int i = 0; i < DT; ++i) {
          uint32_t a[4];
          ldmatrix4_trans(a, sv + chunk_at<D, false>(row, 2 * i + (mi & 1)));
#pragma unroll
          for (int b = 0; b < NB; ++b) mma16816<BF>(acc[i][b], a, pf[t][b][0], pf[t][b][1]);
        }
      }
    }

    const int head = info->head, row0 = info->row0, rows = info->rows, part = info->part;
    const int64_t q0 = info->q0;
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + stage);
    if (++stage == L::kStages) {
      stage = 0;
      phase ^= 1;
    }
    if (!(flags & kLast)) continue;

    // Join the four warps: 2 and 3 into 0 and 1, then 1 into 0.
#pragma unroll
    for (int b = 0; b < NB; ++b) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[b][j] += __shfl_xor_sync(0xffffffffu, l[b][j], d);
      if (Q8) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][b][j] *= vref;
      }
    }
    auto meet = [&]() -> bool {
      __syncwarp();
      if (lane == 0) mbar_arrive(joined);
      const bool ok = mbar_wait_clocked(joined, join_phase);
      join_phase ^= 1;
      if (!ok && lane == 0) raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
      return ok;
    };
    auto give = [&](int to) {
      float *a = merge + to * (kRows * D + 2 * kRows), *s = a + kRows * D;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) a[((i * NB + b) * 4 + j) * 32 + lane] = acc[i][b][j];
        if (r == 0) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[8 * b + 2 * c + j] = m[b][j];
            s[kRows + 8 * b + 2 * c + j] = l[b][j];
          }
        }
      }
    };
    auto take = [&](int from) {
      const float *a = merge + from * (kRows * D + 2 * kRows), *s = a + kRows * D;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float mine[2], theirs[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float om = s[8 * b + 2 * c + j], top = fmaxf(m[b][j], om), ref = top == -INFINITY ? 0.f : top;
          mine[j] = fast_exp2(m[b][j] - ref);
          theirs[j] = fast_exp2(om - ref);
          m[b][j] = top;
          l[b][j] = l[b][j] * mine[j] + s[kRows + 8 * b + 2 * c + j] * theirs[j];
        }
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][b][j] = acc[i][b][j] * mine[j & 1] + a[((i * NB + b) * 4 + j) * 32 + lane] * theirs[j & 1];
      }
    };
    if (warp >= 2) give(warp - 2);
    if (!meet()) return;
    if (warp < 2) take(warp);
    if (!meet()) return;
    if (warp == 1) give(0);
    if (!meet()) return;
    if (warp == 0) take(0);
    if (!meet()) return;  // before the next give
    if (warp != 0) continue;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int col = 8 * b + 2 * c + j, row = row0 + col;
        if (row >= rows) continue;
        if (flags & kWhole) {
          const int t = p.by_group.div(row), g = row - t * p.group;
          if (q0 + t >= p.num_tokens) continue;
          char *out = p.o + (q0 + t) * p.o_row_stride + (static_cast<int64_t>(head) * p.group + g) * p.o_head_stride;
          const float inv = l[b][j] == 0.f ? 0.f : 1.f / l[b][j];
          if (Q8) {
            // dims r W .. + W of each 8 W
#pragma unroll
            for (int i = 0; i < DT; i += 4) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) w[x] = T::pack(acc[i + x][b][j] * inv, acc[i + x][b][2 + j] * inv);
              *reinterpret_cast<uint4 *>(out + ((2 * i / W) * W * 8 + r * W + 2 * i % W) * 2) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            // dims r and r + 8 of each 16: a neighbour's dim beside this lane's
#pragma unroll
            for (int i = 0; i < DT; ++i) {
              const float x = acc[i][b][j] * inv, y = acc[i][b][2 + j] * inv;
              *reinterpret_cast<uint16_t *>(out + (16 * i + r) * 2) = static_cast<uint16_t>(T::pack(x, 0.f));
              *reinterpret_cast<uint16_t *>(out + (16 * i + 8 + r) * 2) = static_cast<uint16_t>(T::pack(y, 0.f));
            }
          }
        } else {
          float *a = p.partials + static_cast<int64_t>(part) * (kRows * D + 2 * kRows), *s = a + kRows * D;
#pragma unroll
          for (int i = 0; i < DT; ++i) {
            if (Q8) {
              *reinterpret_cast<float2 *>(a + col * D + (2 * i / W) * W * 8 + r * W + 2 * i % W) =
                  make_float2(acc[i][b][j], acc[i][b][2 + j]);
            } else {
              a[col * D + 16 * i + r] = acc[i][b][j];
              a[col * D + 16 * i + 8 + r] = acc[i][b][2 + j];
            }
          }
          if (r == 0) {
            s[col] = m[b][j];
            s[kRows + col] = l[b][j];
          }
        }
      }
  }
}

template <typename T, int D, bool Q8, int NB>
__global__ void __launch_bounds__(kThreads, Layout<D, Q8, NB>::kCtas)
    decode_kernel(const __grid_constant__ AttnParams p) {
  using L = Layout<D, Q8, NB>;
  extern __shared__ uint8_t raw[];
  uint8_t *stages = raw + ((128 - (smem_addr(raw) & 127)) & 127);
  float *merge = reinterpret_cast<float *>(stages + L::kStages * L::kStage);
  uint64_t *full = reinterpret_cast<uint64_t *>(stages + L::kStages * L::kStage + L::kMerge);
  uint64_t *empty = full + L::kStages, *joined = empty + L::kStages;
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(full + i, kConsumers * 33);  // the loading warps' copies, and their descriptions
      mbar_init(empty + i, kConsumers);
    }
    mbar_init(joined, kConsumers);
  }
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.items = 0;
  Place place;
  const bool work = find_place<L>(p, place);  // synchronises the block
  pdl_trigger();
  if (!work) {
    if (threadIdx.x == 0) p.meta[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  if (threadIdx.x >= kConsumers * 32) {
    if (L::kCtas == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    load_units<D, Q8, NB>(p, place, stages, full, empty);
  } else {
    // two CTAs: their 2 x 256 x 128 registers, 176 for a computing thread
    if (L::kCtas == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;");
    compute_units<T, D, Q8, NB>(p, place, stages, full, empty, joined, merge);
  }
}

// Joins the parts of a result that began in CTA c - 1 and goes on in CTA c (and
// maybe further): part 2 (c - 1) + 1, then the first parts of the CTAs that
// follow.  One block per (c, query row); 32 lanes per part, parts in turn over
// the warps, then the warps in order.
constexpr int kJoinWarps = 4;
template <typename T, int D, int NB>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ AttnParams p) {
  constexpr int N = D / 32, kRows = 8 * NB;
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

template <typename F>
auto pick(int dtype, int dim, bool q8, int64_t most_rows, F f) {
  auto rows = [&](auto t, auto d, auto q) {
    // 8 query rows a unit where no sequence has more, else 16 (a second block of
    // columns for 4 rows costs 256 8-bit sequences 449 us instead of 340; rows in
    // two units instead of one would read the keys twice)
    if (most_rows <= 8) return f(t, d, q, std::integral_constant<int, 1>{});
    return f(t, d, q, std::integral_constant<int, 2>{});
  };
  auto kind = [&](auto t, auto d) { return q8 ? rows(t, d, std::true_type{}) : rows(t, d, std::false_type{}); };
  auto head = [&](auto t) {
    if (dim == 64) return kind(t, std::integral_constant<int, 64>{});
    if (dim == 128) return kind(t, std::integral_constant<int, 128>{});
    return kind(t, std::integral_constant<int, 256>{});
  };
  return dtype == YL_DTYPE_BF16 ? head(Bf16{}) : head(Fp16{});
}

}  // namespace

int64_t decode_workspace(const yl_paged_attention_args *a, int64_t most_rows) {
  return pick(a->dtype, a->head_dim, a->kv_dtype == YL_KV_E4M3, most_rows, [](auto, auto d, auto q, auto b) {
    using L = Layout<decltype(d)::value, decltype(q)::value, decltype(b)::value>;
    const int64_t ctas = static_cast<int64_t>(sm_count()) * L::kCtas;
    return 16 + ctas * 16 + ctas * 2 * (L::kRows * decltype(d)::value + 2 * L::kRows) * 4;
  });
}

int launch_decode(AttnParams &p, const yl_paged_attention_args *a, int64_t most_rows, cudaStream_t stream) {
  return pick(a->dtype, a->head_dim, a->kv_dtype == YL_KV_E4M3, most_rows, [&](auto t, auto d, auto q, auto b) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value, NB = decltype(b)::value;
    constexpr bool Q8 = decltype(q)::value;
    using L = Layout<D, Q8, NB>;
    const int ctas = sm_count() * L::kCtas;
    p.items = static_cast<int *>(a->workspace);
    p.meta = reinterpret_cast<int4 *>(static_cast<char *>(a->workspace) + 16);
    p.partials = reinterpret_cast<float *>(p.meta + ctas);
    int rc = allow_smem(reinterpret_cast<const void *>(decode_kernel<T, D, Q8, NB>), L::kSmem);
    if (rc != YL_OK) return rc;
    rc = launch_dependent(decode_kernel<T, D, Q8, NB>, dim3(ctas), dim3(kThreads), L::kSmem, stream,
                          "yl_paged_attention launch", p);
    if (rc != YL_OK) return rc;
    return launch_dependent(join_kernel<T, D, NB>, dim3(ctas - 1, static_cast<unsigned>(std::min<int64_t>(most_rows, L::kRows))),
                            dim3(kJoinWarps * 32), 0, stream, "yl_paged_attention launch", p);
  });
}

}  // namespace ylk
