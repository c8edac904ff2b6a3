// Paged attention of sequences with many new tokens (prefill, chunks), for
// sm_100a: both products on the tensor cores, 4 * pairs * head_dim flops per
// query head.
//
// A work item is 2 x 128 query rows of one (sequence, KV head), a row being a
// (new token, head of the group), so a tile of keys serves the whole group.
// One CTA per SM takes items from a counter, the rows that see most first; its
// warps have fixed roles:
//
// * Warps 16-23 load: they gather rows of K and V by page, in tiles of KT tokens,
//   and leave them 16-bit and swizzled in a ring of two stages.  16-bit pools
//   are copied asynchronously; the codes of an 8-bit pool are converted on the
//   way to fp16, which holds every e4m3 value (K's wait for it in shared memory
//   while the tile before is converted, V's in registers).  K's scales, relative
//   to the largest of the tile, are multiplied in: exact for powers of two down to
//   2^-15, two roundings to fp16 for others (factors per column in the softmax
//   instead cost all 8-bit tiles 11 %, for the registers).  The tile's largest goes
//   to the scores as one factor.  V's are multiplied in relative to a reference
//   that changes only when a tile's largest passes 64 times it, when the
//   accumulators are rescaled.
// * Warp 24 issues the products: S = Q K^T per 128 rows (both operands in shared
//   memory), O += P V (P in tensor memory).  The two row tiles alternate, so
//   that one's products run while the other's softmax does.  Warp 25 plans: it
//   finds the items and describes their tiles to the others, some ahead.  (Warps
//   26 and 27 are there for the sharing out of registers.)
// * Warps 0-7 and 8-15 each own a row tile, two threads per row, a half of the
//   columns each: one warp per scheduler would leave the exponentials waiting
//   for one another's latency.  They write Q into shared memory (bf16 queries of
//   an 8-bit pool become fp16 by a power of two per row), then per tile of keys
//   read S once and write the weights over it in 16 bits.  The weights refer to
//   an earlier tile's maximum: that is looked at again, and the row's accumulator
//   rescaled, only where half a row's sum of weights passes 2^15, so that every
//   weight fits fp16; weights are kept times 2^3 there, which puts fp16's
//   smallest numbers 2^-27 below the largest weight of a row that moved.
//
// What bounds it: the products are 4 * 128 * 128 * head_dim flops per row tile
// and key tile, 2,118 cycles for both row tiles at head_dim 128 when nothing else
// runs; a tile takes about 3,850 cycles in the steady state of a 16-bit pool (an
// 8k prompt of 32 heads: 517 us, 1,064 TFLOP/s, 0.65 of the library's measured
// rate) and 4,900 of an 8-bit one (669 us).  The rest is the chain from a score
// product through the softmax to the value product, which the two row tiles
// cover only in part, and for 8-bit pools the conversion.  Masked tiles cost
// about 1,000 cycles more, an item's start and end about 7,000: a window of 1k
// keys has ten tiles per item, two of them masked, and runs at 0.38.  At head_dim
// 256 there is one row tile an item, so products and softmax take turns (8 prompts
// of 128 to 4k tokens: 16-bit 1,147 us, 620 TFLOP/s; 8-bit 1,649), and 88 registers
// are too few for bf16 queries over an 8-bit pool (500 bytes spilled; 178 at 128).
//
// Only tiles that some row does not see in full are masked; in those, infinities
// and NaN of V are zeroed as they are loaded and reported to the rows that see
// them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cstdint>

#include "attend_device.cuh"
#include "tcgen05.cuh"

namespace ylk {
namespace {

constexpr int kSoftmaxWarps = 16, kLoadWarps = 8;
constexpr int kThreads = (kSoftmaxWarps + kLoadWarps + 4) * 32;
constexpr int kLoadThreads = kLoadWarps * 32;
constexpr int kTileThreads = 256;  // softmax threads of a row tile
constexpr int kStages = 2;  // of K, and of V
constexpr int kInfos = 4;   // descriptions of tiles: one is read until the tile's values are used up
constexpr float kMost = 32768.f;  // sum of weights of half a row, lift included, above which they are looked at again
constexpr float kMaxRatio = 64.f; // of a V scale to the reference

constexpr int kHeader = 12288;  // bytes of Shared

template <int D>
struct Shape {
  static constexpr int kQTiles = D == 256 ? 1 : 2;  // 128-row tiles of an item
  static constexpr int kKT = D == 256 ? 64 : 128;   // tokens of a key tile
  static constexpr int kRows = 128 * kQTiles;
  static constexpr int kQBytes = 128 * D * 2;       // one row tile
  static constexpr int kKVBytes = kKT * D * 2;      // K or V of a stage
  static constexpr int kRaw = kKT * D;              // codes of a tile of K
  static constexpr int kSmem = kQTiles * kQBytes + 2 * kStages * kKVBytes + kHeader + 1024;  // without kRaw
  static constexpr uint32_t kS = 0;    // tensor memory columns: S of tile w at w * kKT
  static constexpr uint32_t kO = 256;  // O of tile w at kO + w * D
};

// What the loading warps say about a tile of keys.
struct TileInfo {
  float key;         // factor of the scores
  float move;        // factor of the accumulators before this tile
  float value;       // what the accumulators are multiples of, from this tile on
  int base;          // position of the first token
  int edge;          // some row does not see every token
  int live;          // row tiles of the item; 0: there are no more tiles
  int last;          // of its item
  uint32_t valid[4]; // tokens with a good page
  uint32_t ghost[4]; // edge tiles: tokens whose V had an infinity or NaN
};

// The planning warp's word on a tile.
struct Plan {
  int base, cnt;            // first position and tokens of it
  int e0, head;             // of the sequence; KV head
  int first_pos, last_pos;  // of the item's queries
  int live;                 // row tiles of the item; 0: there are no more tiles
  int flags;                // kFirst | kLast of its item
};
constexpr int kFirst = 1, kLast = 2, kPlans = 4;

// And on an item.
struct ItemInfo {
  int tiles;  // 0: there are no more items
  int q0, first;  // of its sequence: row of q and o, position
  int head, row0, rows;
};

struct Shared {
  uint64_t k_full[kStages], v_full[kStages], k_empty[kStages], v_empty[kStages];
  uint64_t item_full[2], item_empty[2], plan_full[kPlans], plan_empty[kPlans];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t described[2];  // a row tile has read the last of an item's descriptions
  uint64_t drained;
  uint32_t tmem;
  float top[2][2][kLoadWarps];     // [parity][K, V][loading warp]: largest scales
  uint32_t valid[2][4];            // [parity]: tokens with a good page
  TileInfo tile[kInfos];
  ItemInfo item[2];
  Plan plan[kPlans];
  int64_t offset[2][128];          // [parity]: byte offset of a token's head row
  uint32_t ratio[2][2][128];       // [parity][K, V]: scale over the reference, two halves
  float rows[2][2][128];           // [row tile][half of the columns]: a row's maximum or sum
  int64_t row_at[2][2][128];       // [row tile][q, o]: byte offset of a row, -1 for none
};
static_assert(sizeof(Shared) <= kHeader, "shared header");

struct Item {
  Seq seq;
  int head;  // KV head
  int row0;  // first query row
  int rows;  // query rows of the sequence and KV head
  Span span;
  int first_pos, last_pos;  // positions of the item's first and last query
  int head_tiles, tiles;
};

// Finds items by number, in increasing order, by a whole warp: 32 sequences at a
// time.  A sequence's items come with the last rows first (they see most).
template <int D>
class Walker {
 public:
  __device__ __forceinline__ Walker(const AttnParams &p) : p_(p) {}
  __device__ __forceinline__ bool seek(int64_t n, Item &out) {
    const int lane = threadIdx.x & 31;
    while (base_ < p_.batch) {
      if (!loaded_) {
        units_ = 0;
        if (base_ + lane < p_.batch) {
          seq_ = load_seq(p_, base_ + lane, false);
          const int64_t rows = static_cast<int64_t>(seq_.fresh) * p_.group;
          if (rows > p_.max_rows) units_ = (rows + Shape<D>::kRows - 1) / Shape<D>::kRows * p_.heads;
        }
        scan_ = units_;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, scan_, d);
          if (lane >= d) scan_ += y;
        }
        loaded_ = true;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before_ + scan_ > n);
      if (past != 0) {
        const int at = __ffs(past) - 1;
        Seq s;
        s.q0 = __shfl_sync(0xffffffffu, seq_.q0, at);
        s.fresh = __shfl_sync(0xffffffffu, seq_.fresh, at);
        s.first = __shfl_sync(0xffffffffu, seq_.first, at);
        s.e0 = __shfl_sync(0xffffffffu, seq_.e0, at);
        s.total = __shfl_sync(0xffffffffu, seq_.total, at);
        const int64_t units = __shfl_sync(0xffffffffu, units_, at);
        const int64_t start = before_ + __shfl_sync(0xffffffffu, scan_, at) - units;
        const int k = static_cast<int>(n - start);
        out.seq = s;
        out.head = k % p_.heads;
        out.row0 = (static_cast<int>(units / p_.heads) - 1 - k / p_.heads) * Shape<D>::kRows;
        out.rows = s.fresh * p_.group;
        const int t0 = p_.by_group.div(out.row0);
        const int t1 = p_.by_group.div(min(out.rows, out.row0 + Shape<D>::kRows) - 1) + 1;
        out.span = span_of(p_, s, t0, t1);
        out.first_pos = max(s.first + t0, -1);  // (-1, like all below it, sees nothing)
        out.last_pos = max(s.first + t1 - 1, -1);
        constexpr int KT = Shape<D>::kKT;
        out.head_tiles = (out.span.head + KT - 1) / KT;
        out.tiles = max(1, out.head_tiles + (out.span.end - out.span.low + KT - 1) / KT);
        return true;
      }
      before_ += __shfl_sync(0xffffffffu, scan_, 31);
      base_ += 32;
      loaded_ = false;
    }
    return false;
  }

 private:
  const AttnParams &p_;
  int base_ = 0;
  bool loaded_ = false;
  int64_t before_ = 0, units_ = 0, scan_ = 0;
  Seq seq_{};
};

__device__ __forceinline__ bool wait_or_report(const AttnParams &p, uint64_t *bar, uint32_t parity) {
  if (mbar_wait_clocked(bar, parity)) return true;
  raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
  return false;
}
// The same answer for the whole warp.
__device__ __forceinline__ bool warp_wait(const AttnParams &p, uint64_t *bar, uint32_t parity) {
  const bool ok = mbar_wait_clocked(bar, parity);
  if (!ok) raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
  return __all_sync(0xffffffffu, ok);
}
// Barrier of the loading warps; whether all of them passed true.
__device__ __forceinline__ bool load_barrier(bool fine) {
  uint32_t all;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 q, %1, 0;\n"
      "barrier.cta.red.and.pred p, 1, 256, q;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(fine))
      : "memory");
  return all != 0;
}

// Barrier of a row tile's softmax threads; whether any of them passed true.
__device__ __forceinline__ bool tile_barrier(int w, bool any) {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 q, %1, 0;\n"
      "barrier.cta.red.or.pred p, %2, 256, q;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(any)), "r"(2 + w)
      : "memory");
  return r != 0;
}

// ---------------------------------------------------------------------------
// Loading warps
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <bool BF>
__device__ __forceinline__ uint32_t drop_nonfinite(uint32_t &w) {
  const uint32_t mask = __vcmpgeu2(w & 0x7fff7fffu, BF ? 0x7f807f80u : 0x7c007c00u);
  w &= ~mask;
  return mask;
}

__device__ __forceinline__ void sts128(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Shared-memory position of 16-byte chunk c of row r of a tile of ROWS rows.
template <int ROWS>
__device__ __forceinline__ uint32_t swizzled(int r, int c) {
  return (c >> 3) * (ROWS * 128) + r * 128 + (((c ^ r) & 7) << 4);
}

// Each thread looks up one token of a tile: its page id two tiles ahead, the
// page's scales one tile ahead.
template <typename T, int D, bool Q8>
__device__ __forceinline__ void load_tiles(const AttnParams &p, Shared *sh, uint8_t *kv, uint8_t *raw) {
  using S = Shape<D>;
  constexpr int KT = S::kKT;
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;
  constexpr int kNone = -0x7fffffff, kNoEntry = -0x7ffffffe;  // not a token of the tile; no such entry
  const int tid = threadIdx.x - kSoftmaxWarps * 32, lane = tid & 31, warp = tid >> 5;
  auto page_of = [&](const Plan &t) {
    if (tid >= KT || tid >= t.cnt) return kNone;
    const int64_t e = static_cast<int64_t>(t.e0) + p.by_page.div(t.base + tid);
    return e >= 0 && e < p.indices_cap ? __ldg(p.kv_indices + e) : kNoEntry;
  };
  auto good = [&](int page) { return page >= 0 && page < p.num_pages; };
  auto scales_of = [&](const Plan &t, int page, float &ks, float &vs) {
    ks = vs = 0.f;
    if (Q8 && good(page)) {
      const int64_t sc = static_cast<int64_t>(page) * p.scale_page_stride + t.head * p.scale_head_stride;
      ks = __ldg(p.scale[0] + sc);
      vs = __ldg(p.scale[1] + sc);
    }
  };
  // plan u, waited for; the plans behind the last tile's stay unread
  auto plan = [&](uint32_t u) -> const Plan & { return sh->plan[u % kPlans]; };
  auto planned = [&](uint32_t u) { return warp_wait(p, &sh->plan_full[u % kPlans], u / kPlans & 1); };
  const bool begun = planned(0);
  bool more0 = begun && plan(0).live != 0;
  const bool early = begun && (!more0 || planned(1));
  bool more1 = more0 && early && plan(1).live != 0;
  if (!load_barrier(early)) return;  // all of them, or none
  int page0 = more0 ? page_of(plan(0)) : kNone, page1 = more1 ? page_of(plan(1)) : kNone;
  float ks0 = 0.f, vs0 = 0.f;
  if (more0) scales_of(plan(0), page0, ks0, vs0);
  // where the rows of tile u are, for all threads
  auto place = [&](uint32_t u, int page) {
    const Plan &t = plan(u);
    int64_t off = -1;
    if (good(page)) {
      const int pos = t.base + tid;
      off = static_cast<int64_t>(page) * p.page_stride +
            static_cast<int64_t>(pos - static_cast<int>(p.by_page.div(pos)) * p.page_size) * p.slot_stride +
            t.head * p.head_stride;
    } else if (page != kNone) {
      raise_deverr(p.error_word, page == kNoEntry ? YL_DEVERR_INDICES_CAP : YL_DEVERR_PAGE_RANGE);
    }
    if (tid < KT) sh->offset[u & 1][tid] = off;
    const uint32_t ok = __ballot_sync(0xffffffffu, off >= 0);
    if (lane == 0 && warp * 32 < KT) sh->valid[u & 1][warp] = ok;
  };
  constexpr int CH = D * (Q8 ? 1 : 2) / 16;    // 16-byte chunks of a token's head row
  constexpr int STEP = kLoadThreads / CH;      // rows of one pass of the threads
  constexpr int PER = KT / STEP;               // chunks of a thread
  const int c = tid % CH, r0 = tid / CH;
  // K's codes of tile u, each thread's chunks into its own places of `raw`
  const uint32_t mine = smem_addr(raw) + tid * 16;
  auto fetch_keys = [&](uint32_t u) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t o = sh->offset[u & 1][r0 + i * STEP];
      cp_async16(mine + i * kLoadThreads * 16, p.kv[0] + (o >= 0 ? o + c * 16 : 0), o >= 0);
    }
  };
  if (more0) {
    place(0, page0);
    load_barrier(true);
    if (Q8) fetch_keys(0);
  }
  float value = 0.f;  // reference of V's scales
  bool lost = false;  // a wait gave up: the next barrier ends all of them
  uint32_t used = 0;
  for (; more0; ++used) {
    const int stage = used % kStages, par = used & 1;
    const uint32_t phase = (used / kStages & 1) ^ 1;
    bool fine = !more1 || planned(used + 2);
    const bool more2 = fine && more1 && plan(used + 2).live != 0;
    const int page2 = more2 ? page_of(plan(used + 2)) : kNone;
    float ks1 = 0.f, vs1 = 0.f;
    if (more1) scales_of(plan(used + 1), page1, ks1, vs1);
    const Plan &t0 = plan(used);

    if (Q8) {
      // (positive numbers are ordered like their bits; a scale that is no number is
      // left out here and reaches the rows that see its token with its codes)
      auto largest = [](float s) {
        const uint32_t b = __float_as_uint(s);
        return __uint_as_float(__reduce_max_sync(0xffffffffu, b < 0x7f800000u ? b : 0u));
      };
      const float ktop = largest(ks0), vtop = largest(vs0);
      if (lane == 0) {
        sh->top[par][0][warp] = ktop;
        sh->top[par][1][warp] = vtop;
      }
    }
    load_barrier(true);
    if (more1) place(used + 1, page1);  // (nobody reads the tile before this one's places any more)
    float key = 1.f, move = 1.f;
    if (t0.flags & kFirst) value = Q8 ? 0.f : 1.f;
    if (Q8) {
      float ktop = 0.f, vtop = 0.f;
#pragma unroll
      for (int k = 0; k < KT / 32; ++k) {
        ktop = fmaxf(ktop, sh->top[par][0][k]);
        vtop = fmaxf(vtop, sh->top[par][1][k]);
      }
      if (ktop > 0.f) key = ktop;
      if (vtop > value * kMaxRatio) {
        move = value / vtop;
        value = vtop;
      }
      if (tid < KT) {
        const float rk = ks0 / key, rv = vs0 / (value > 0.f ? value : 1.f);
        sh->ratio[par][0][tid] = Fp16::pack(rk, rk);
        sh->ratio[par][1][tid] = Fp16::pack(rv, rv);
      }
    }
    // a tile with a bad page is masked like one that some row sees in part
    uint32_t all = 0xffffffffu;
#pragma unroll
    for (int k = 0; k < KT / 32; ++k) all &= sh->valid[par][k];
    const bool edge = all != 0xffffffffu || t0.base + KT - 1 > t0.first_pos ||
                      (p.window > 0 && t0.base <= t0.last_pos - p.window && t0.base + KT > p.sinks);
    const uint32_t sk = smem_addr(kv + stage * 2 * S::kKVBytes), sv = sk + S::kKVBytes;
    uint4 w[Q8 ? PER : 1];
    if (Q8) {  // V's codes are on their way before K is converted
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int64_t o = sh->offset[par][r0 + i * STEP];
        w[i] = ldg128_if(p.kv[1] + o + c * 16, o >= 0);
      }
    }
    // K's previous tile of this stage is used up; V's is waited for behind K
    fine = fine && !lost && wait_or_report(p, &sh->k_empty[stage], phase);
    TileInfo *info = &sh->tile[used % kInfos];
    if (tid == 0) {
      info->key = key;
      info->move = move;
      info->value = value;
      info->base = t0.base;
      info->edge = edge;
      info->live = t0.live;
      info->last = t0.flags & kLast;
    }
    if (tid < KT / 32) {
      info->valid[tid] = sh->valid[par][tid];
      info->ghost[tid] = 0;
    }
    if (!load_barrier(fine)) break;
    if (lane == 0) mbar_arrive(&sh->plan_empty[used % kPlans]);  // (every thread has read it)

    if (Q8) {
      auto convert = [&](const uint32_t (&x)[4], int r, int kv_i) {
        const uint32_t ratio = sh->ratio[par][kv_i][r];
        uint32_t y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          y[2 * k] = mul_half2(e4m3x2_to_half2(static_cast<uint16_t>(x[k])), ratio);
          y[2 * k + 1] = mul_half2(e4m3x2_to_half2(static_cast<uint16_t>(x[k] >> 16)), ratio);
        }
        if (kv_i == 1 && edge) {
          uint32_t any = 0;
#pragma unroll
          for (int k = 0; k < 8; ++k) any |= drop_nonfinite<false>(y[k]);
          if (any) atomicOr(&info->ghost[r >> 5], 1u << (r & 31));
        }
        const uint32_t at = kv_i ? sv : sk;
        sts128(at + swizzled<KT>(r, 2 * c), y[0], y[1], y[2], y[3]);
        sts128(at + swizzled<KT>(r, 2 * c + 1), y[4], y[5], y[6], y[7]);
      };
      cp_async_wait_all();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        uint32_t x[4];
        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                     : "r"(mine + i * kLoadThreads * 16)
                     : "memory");
        convert(x, r0 + i * STEP, 0);
      }
      fence_to_async();
      mbar_arrive(&sh->k_full[stage]);
      if (more1) fetch_keys(used + 1);  // on their way while V is converted
      lost = !wait_or_report(p, &sh->v_empty[stage], phase);
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        convert(x, r0 + i * STEP, 1);
      }
      fence_to_async();
      mbar_arrive(&sh->v_full[stage]);
    } else {
#pragma unroll
      for (int kv_i = 0; kv_i < 2; ++kv_i) {
        if (kv_i == 1) lost = !wait_or_report(p, &sh->v_empty[stage], phase);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const int r = r0 + i * STEP;
          const int64_t o = sh->offset[par][r];
          cp_async16((kv_i ? sv : sk) + swizzled<KT>(r, c), p.kv[kv_i] + (o >= 0 ? o + c * 16 : 0), o >= 0);
        }
        if (kv_i == 0 || !edge) {
          cp_async_arrive(smem_addr(kv_i ? &sh->v_full[stage] : &sh->k_full[stage]));  // when they have landed
        } else {
          cp_async_wait_all();
#pragma unroll 1
          for (int i = 0; i < PER; ++i) {  // the chunks that this thread copied
            const int r = r0 + i * STEP;
            const uint32_t at = sv + swizzled<KT>(r, c);
            uint32_t x[4];
            asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
            uint32_t any = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) any |= drop_nonfinite<BF>(x[k]);
            if (any) {
              atomicOr(&info->ghost[r >> 5], 1u << (r & 31));
              sts128(at, x[0], x[1], x[2], x[3]);
            }
          }
          mbar_arrive(&sh->v_full[stage]);
        }
      }
    }
    more0 = more1;
    more1 = more2;
    page0 = page1;
    page1 = page2;
    ks0 = ks1;
    vs0 = vs1;
  }
  cp_async_wait_all();
  // no more: an empty tile says so, in its turn
  if (wait_or_report(p, &sh->k_empty[used % kStages], (used / kStages & 1) ^ 1)) {
    if (tid == 0) sh->tile[used % kInfos].live = 0;
    mbar_arrive(&sh->k_full[used % kStages]);
  }
}

// ---------------------------------------------------------------------------
// Planning warp
// ---------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ void plan_tiles(const AttnParams &p, Shared *sh) {
  constexpr int KT = Shape<D>::kKT;
  const int lane = threadIdx.x & 31;
  Walker<D> walker(p);
  Item it{};
  uint32_t items = 0, used = 0;
  int64_t n = blockIdx.x;
  for (;; ++items) {
    const bool more = walker.seek(n, it);
    if (!warp_wait(p, &sh->item_empty[items & 1], (items >> 1 & 1) ^ 1)) return;
    if (lane == 0) {
      sh->item[items & 1] = ItemInfo{more ? it.tiles : 0, it.seq.q0, it.seq.first, it.head, it.row0, it.rows};
      mbar_arrive(&sh->item_full[items & 1]);
      if (more) n = static_cast<int64_t>(gridDim.x) + atomicAdd(p.items, 1);
    }
    n = __shfl_sync(0xffffffffu, n, 0);
    // its queries on their way into the L2 cache
    if (more)
      for (int i = lane; i < Shape<D>::kRows * (D / 64); i += 32) {
        const int row = it.row0 + i / (D / 64), t = p.by_group.div(row);
        if (row < it.rows && it.seq.q0 + static_cast<int64_t>(t) < p.num_tokens)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(
              p.q + (it.seq.q0 + static_cast<int64_t>(t)) * p.q_row_stride +
              (static_cast<int64_t>(it.head) * p.group + (row - t * p.group)) * p.q_head_stride + i % (D / 64) * 128));
      }
    const int live = more ? min(Shape<D>::kQTiles, (it.rows - it.row0 + 127) / 128) : 0;
    for (int j = 0; j < (more ? it.tiles : 1); ++j, ++used) {
      const int slot = used % kPlans;
      if (!warp_wait(p, &sh->plan_empty[slot], (used / kPlans & 1) ^ 1)) return;
      if (lane == 0) {
        const bool in_head = j < it.head_tiles;
        Plan t;
        t.base = (in_head ? 0 : it.span.low) + (in_head ? j : j - it.head_tiles) * KT;
        t.cnt = min(KT, (in_head ? it.span.head : it.span.end) - t.base);
        t.e0 = it.seq.e0;
        t.head = it.head;
        t.first_pos = it.first_pos;
        t.last_pos = it.last_pos;
        t.live = live;
        t.flags = (j == 0 ? kFirst : 0) | (j == it.tiles - 1 ? kLast : 0);
        sh->plan[slot] = t;
        mbar_arrive(&sh->plan_full[slot]);
      }
      __syncwarp();
    }
    if (!more) return;
  }
}

// ---------------------------------------------------------------------------
// Product warp
// ---------------------------------------------------------------------------
template <typename T, int D, bool Q8>
__device__ __forceinline__ void issue_products(const AttnParams &p, Shared *sh, uint8_t *q, uint8_t *kv) {
  using S = Shape<D>;
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;
  constexpr int KT = S::kKT;
  constexpr uint32_t kScores = f16_product(BF, 128, KT, false), kValues = f16_product(BF, 128, D, true);
  const uint32_t tmem = sh->tmem, sq = smem_addr(q), skv = smem_addr(kv);
  uint32_t queries[2] = {0, 0}, weights[2] = {0, 0};  // waits on q_full and p_full so far
  // scores of a tile for row tile w; `done`: the last row tile's, K is used up
  auto scores = [&](int w, uint32_t tile, bool done) {
    const uint64_t a = tile_desc(sq + w * S::kQBytes, 16);
    const uint64_t b = tile_desc(skv + (tile % kStages) * 2 * S::kKVBytes, 16);
    if (elect_one()) {
#pragma unroll
      for (int s = 0; s < D / 16; ++s)  // (addresses count in 16 bytes)
        mma_ss(tmem + S::kS + w * KT, a + ((s / 4) * (128 * 128) + (s % 4) * 32) / 16,
               b + ((s / 4) * (KT * 128) + (s % 4) * 32) / 16, kScores, s > 0);
      mma_commit(&sh->s_full[w]);
      if (done) mma_commit(&sh->k_empty[tile % kStages]);
    }
    __syncwarp();
  };
  bool first = true;
  for (uint32_t tile = 0;; ++tile) {
    const int stage = tile % kStages;
    const uint32_t phase = tile / kStages & 1;
    const TileInfo *info = &sh->tile[tile % kInfos];
    if (first) {  // of its item
      if (!warp_wait(p, &sh->k_full[stage], phase)) break;
      const int live = info->live;
      if (live == 0) break;
      fence_to_async();  // (asynchronous copies of a 16-bit pool arrive without one)
      bool ok = true;
      for (int w = 0; w < live && ok; ++w) {
        ok = warp_wait(p, &sh->q_full[w], queries[w]++ & 1);
        if (!ok) break;
        tc_fence_after();
        scores(w, tile, w == live - 1);
      }
      // A row tile that this item lacks may still be at the end of an item before,
      // whose last tile's description must not be written over: that is done for
      // the fourth tile behind it, once the keys of the second are used up, by a
      // product that is behind this wait.  (The row tile's next item is too, so the
      // barrier is in this phase or just past it.)
      for (int w = live; w < S::kQTiles && ok; ++w)
        ok = queries[w] == 0 || warp_wait(p, &sh->described[w], (queries[w] - 1) & 1);
      if (!ok) break;
    }
    const int live = info->live;
    const bool last = info->last != 0;
    if (!warp_wait(p, &sh->v_full[stage], phase)) break;
    if (!last && !warp_wait(p, &sh->k_full[(tile + 1) % kStages], (tile + 1) / kStages & 1)) break;
    fence_to_async();
    bool ok = true;
    for (int w = 0; w < live && ok; ++w) {
      ok = warp_wait(p, &sh->p_full[w], weights[w]++ & 1);
      if (!ok) break;
      tc_fence_after();
      const uint64_t b = tile_desc(skv + stage * 2 * S::kKVBytes + S::kKVBytes, KT * 128);
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < KT / 16; ++s)
          mma_ts(tmem + S::kO + w * D, tmem + S::kS + w * KT + s * 8, b + s * (2048 / 16), kValues, !first || s > 0);
        if (w == live - 1) mma_commit(&sh->v_empty[stage]);
        if (last) mma_commit(&sh->o_full[w]);
      }
      __syncwarp();
      if (last) continue;
      scores(w, tile + 1, w == live - 1);
    }
    if (!ok) break;
    first = last;
  }
  // nothing of this CTA is in flight when its tensor memory goes
  if (elect_one()) mma_commit(&sh->drained);
  __syncwarp();
  warp_wait(p, &sh->drained, 0);
}

// ---------------------------------------------------------------------------
// Softmax warps: row tile w, half of the columns, one row per thread
// ---------------------------------------------------------------------------
// Pairs of floats in packed arithmetic.
__device__ __forceinline__ uint64_t pair2(uint32_t a, uint32_t b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) { return pair2(__float_as_uint(a), __float_as_uint(b)); }
__device__ __forceinline__ void unpack2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The lowest n bits, n of any sign.
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// This half row's accumulator times a factor (rare: the reference of the weights
// or of V's scales moved).
template <int COLUMNS>
__device__ __forceinline__ void rescale(uint32_t at, float factor) {
#pragma unroll 1
  for (int k = 0; k < COLUMNS / 32; ++k) {
    uint32_t x[32];
    tmem_ld32(at + 32 * k, x);
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * factor);
    tmem_st32(at + 32 * k, x);
  }
}

template <typename T, int D, bool Q8>
__device__ __forceinline__ void softmax_rows(const AttnParams &p, Shared *sh, uint8_t *q, int w, int half) {
  using S = Shape<D>;
  constexpr int KT = S::kKT, C = KT / 2, DC = D / 2;  // columns of S and of O of this half
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;
  constexpr float kLift = BF ? 0.f : 3.f;
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int r = warp * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t ts = sh->tmem + lanes + S::kS + w * KT + half * C;      // scores of this half
  const uint32_t tp = sh->tmem + lanes + S::kS + w * KT + half * C / 2;  // weights, two to a column
  const uint32_t to = sh->tmem + lanes + S::kO + w * D + half * DC;
  const uint32_t sq = smem_addr(q) + w * S::kQBytes;
  float *mine = &sh->rows[w][half][r], *other = &sh->rows[w][half ^ 1][r];
  uint32_t used = 0, waits = 0, done = 0;
  // After a wait that gave up a thread waits no more, but meets its row tile's
  // barriers until all of them leave together, at the next item.
  bool lost = false;
  auto wait = [&](uint64_t *bar, uint32_t parity) { lost = lost || !warp_wait(p, bar, parity); };
  for (uint32_t items = 0;; ++items) {
    wait(&sh->item_full[items & 1], items >> 1 & 1);
    if (tile_barrier(w, lost)) return;
    const ItemInfo it = sh->item[items & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->item_empty[items & 1]);
    if (it.tiles == 0) return;
    if (w >= S::kQTiles || it.row0 + w * 128 >= it.rows) {  // an item without this row tile
      used += it.tiles;
      continue;
    }
    const int pos = max(it.first + static_cast<int>(p.by_group.div(min(it.row0 + w * 128 + r, it.rows - 1))), -1);
    // Rows move between global and shared memory in whole: 16-byte chunk
    // `chunk` of rows r0, r0 + STEP, .. is this thread's.
    constexpr int CH = D / 8, STEP = kTileThreads / CH, PER = 128 / STEP;
    const int tid = threadIdx.x & (kTileThreads - 1), chunk = tid % CH, r0 = tid / CH;
    {  // their places: row r of the row tile in q (half 0) or o (half 1)
      const int row = it.row0 + w * 128 + r, t = p.by_group.div(row);
      const int64_t token = it.q0 + static_cast<int64_t>(t), head = static_cast<int64_t>(it.head) * p.group + (row - t * p.group);
      const bool has = row < it.rows && token < p.num_tokens;
      sh->row_at[w][half][r] = !has ? -1 : half ? token * p.o_row_stride + head * p.o_head_stride
                                                : token * p.q_row_stride + head * p.q_head_stride;
    }
    tile_barrier(w, false);
    // the queries, 16-bit and swizzled
    float coef = p.scale_log2;
    {
      uint4 x[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int64_t at = sh->row_at[w][0][r0 + i * STEP];
        x[i] = at >= 0 ? __ldg(reinterpret_cast<const uint4 *>(p.q + at) + chunk) : make_uint4(0, 0, 0, 0);
      }
      if (Q8 && std::is_same<T, Bf16>::value) {
#pragma unroll
        for (int i = 0; i < PER; i += 2) {  // two rows' largest elements in one word
          auto largest = [](const uint4 &v) {
            const uint32_t b = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu),
                                        __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
            return max(b & 0xffffu, b >> 16);
          };
          uint32_t big = largest(x[i]) | largest(x[i + 1]) << 16;
#pragma unroll
          for (int d = CH / 2; d > 0; d >>= 1) big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, d));
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int e = min(max(static_cast<int>((k ? big >> 16 : big & 0xffffu) >> 7), 1), 253);  // biased exponent
            const float up = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
            if (chunk == 0) sh->rows[w][0][r0 + (i + k) * STEP] = __uint_as_float(static_cast<uint32_t>(e) << 23);
            auto turn = [&](uint32_t &v) {
              const float2 f = Bf16::unpack(v);
              v = Fp16::pack(f.x * up, f.y * up);
            };
            turn(x[i + k].x);
            turn(x[i + k].y);
            turn(x[i + k].z);
            turn(x[i + k].w);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < PER; ++i) sts128(sq + swizzled<128>(r0 + i * STEP, chunk), x[i].x, x[i].y, x[i].z, x[i].w);
      fence_to_async();
      tc_fence_before();  // the previous item's accumulators are read
      mbar_arrive(&sh->q_full[w]);
      if (Q8 && std::is_same<T, Bf16>::value) {
        tile_barrier(w, false);
        coef *= sh->rows[w][0][r];
        tile_barrier(w, false);  // before the array's next use
      }
    }

    // the columns of word k of a tile that this row sees
    auto seen = [&](const TileInfo *info, int word) {
      const int base = info->base + 32 * word;
      uint32_t see = info->valid[word] & low_bits(pos - base + 1);
      if (p.window > 0) see &= ~low_bits(pos - p.window - base + 1) | low_bits(p.sinks - base);
      return see;
    };
    bool ghostly = false;  // a value that this row sees was no number
    auto look_back = [&](uint32_t tile) {  // at an edge tile whose values are loaded by now
      const TileInfo *info = &sh->tile[tile % kInfos];
#pragma unroll
      for (int k = 0; k < C / 32; ++k)
        if (info->ghost[half * (C / 32) + k] & seen(info, half * (C / 32) + k)) ghostly = true;
    };
    bool edge = false;
    float m = -INFINITY, l = 0.f, value = 1.f;  // l: this half's sum
    for (int j = 0; j < it.tiles; ++j, ++used) {
      wait(&sh->s_full[w], waits++ & 1);  // (issued behind the tile's description)
      tc_fence_after();
      const TileInfo *info = &sh->tile[used % kInfos];
      // Kept a normal number: a zero row's factor is scale_log2 * 2^-126, and times
      // a K scale of 2^-22 it would be 0, which times the -inf of a hidden column
      // is no number.  (A row's scores are at most 2^18 times the factor, so the
      // smallest normal one stands for all below it; the largest, so that 0 times
      // it stays 0.)
      const float c = Q8 ? fminf(fmaxf(coef * info->key, FLT_MIN), FLT_MAX) : coef;
      float factor = info->move;
      if (edge) look_back(used - 1);  // (the scores' products were issued behind its values')
      edge = info->edge != 0;
      value = info->value;
      auto hide = [&](uint32_t (&x)[32], int k) {  // the columns of chunk k that this row does not see
        const uint32_t see = seen(info, half * (C / 32) + k);
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (!(see & (1u << i))) x[i] = 0xff800000u;  // -inf
      };
      uint32_t y[C / 2];  // the weights, not written before every thread of the row tile has read its scores
      float sum;
      const uint64_t c2 = pack2(c, c);
      auto weigh = [&]() {
        const float off = kLift - (m == -INFINITY ? 0.f : m);
        const uint64_t off2 = pack2(off, off);
        uint64_t sums[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < C / 32; ++k) {
          uint32_t x[32];
          tmem_ld32(ts + 32 * k, x);
          if (edge) hide(x, k);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float u, v;
            unpack2(fma2(pair2(x[2 * i], x[2 * i + 1]), c2, off2), u, v);
            u = fast_exp2(u);
            v = fast_exp2(v);
            sums[i & 1] = add2(sums[i & 1], pack2(u, v));
            y[16 * k + i] = BF ? Bf16::pack(u, v) : Fp16::pack(u, v);
          }
        }
        float s0, s1;
        unpack2(add2(sums[0], sums[1]), s0, s1);
        sum = s0 + s1;
      };
      // First with the reference as it stands: the sum of the weights tells whether
      // any of them passes kMost, or is no number.
      bool again = j == 0;
      if (!again) {
        again = __any_sync(0xffffffffu, m == -INFINITY);
        if (!again) {
          weigh();
          again = !(sum <= kMost);
        }
        again = tile_barrier(w, again);
      }
      if (again) {
        // Else, and for the first tile, the maximum first; rows whose weights would
        // pass 1 take it as their reference, all of them while the tile is here:
        // when only weights above 2^8 moved it, some row came back at every third
        // tile of scores with a spread of tens.
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < C / 32; ++k) {
          uint32_t x[32];
          tmem_ld32(ts + 32 * k, x);
          if (edge) hide(x, k);
          float tops[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 16; ++i)
            tops[i & 1] = fmaxf(tops[i & 1], fmaxf(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])));
          top = fmaxf(top, fmaxf(tops[0], tops[1]));
        }
        *mine = top;
        tile_barrier(w, false);
        top = fmaxf(top, *other) * c;
        if (top > m) {
          const float f = fast_exp2(m - top);
          m = top;
          l *= f;
          factor *= f;
        }
        weigh();
        tile_barrier(w, false);  // before the first weight over scores, and before the next maximum
      }
      l += sum;
      if constexpr (C == 64)
        tmem_st32(tp, y);
      else
        tmem_st16(tp, y);
      if (j > 0 && __any_sync(0xffffffffu, factor != 1.f)) rescale<DC>(to, factor);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&sh->p_full[w]);
    }

    wait(&sh->o_full[w], done++ & 1);
    tc_fence_after();
    if (edge) look_back(used - 1);
    *mine = ghostly ? NAN : l;
    tile_barrier(w, false);
    if (tid == 0) mbar_arrive(&sh->described[w]);
    l = (ghostly ? NAN : l) + *other;
    const float inv = l == 0.f ? 0.f : value / l;
    // through the shared memory of the queries, which are used up
#pragma unroll
    for (int k = 0; k < DC / 32; ++k) {
      uint32_t x[32];
      tmem_ld32(to + 32 * k, x);
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        uint32_t y[4];
#pragma unroll
        for (int a = 0; a < 4; ++a)
          y[a] = T::pack(__uint_as_float(x[i + 2 * a]) * inv, __uint_as_float(x[i + 2 * a + 1]) * inv);
        sts128(sq + swizzled<128>(r, half * (DC / 8) + 4 * k + i / 8), y[0], y[1], y[2], y[3]);
      }
    }
    tile_barrier(w, false);
    if (lost) continue;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t at = sh->row_at[w][1][r0 + i * STEP];
      uint32_t y[4];
      asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(y[0]), "=r"(y[1]), "=r"(y[2]), "=r"(y[3])
                   : "r"(sq + swizzled<128>(r0 + i * STEP, chunk)));
      if (at >= 0) *(reinterpret_cast<uint4 *>(p.o + at) + chunk) = make_uint4(y[0], y[1], y[2], y[3]);
    }
  }
}

template <typename T, int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 1) prefill_kernel(const __grid_constant__ AttnParams p) {
  using S = Shape<D>;
  extern __shared__ uint8_t raw[];
  uint8_t *q = raw + ((1024 - (smem_addr(raw) & 1023)) & 1023);
  uint8_t *kv = q + S::kQTiles * S::kQBytes;
  Shared *sh = reinterpret_cast<Shared *>(kv + 2 * kStages * S::kKVBytes);
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&sh->k_full[i], kLoadThreads);
      mbar_init(&sh->v_full[i], kLoadThreads);
      mbar_init(&sh->k_empty[i], 1);
      mbar_init(&sh->v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh->q_full[i], kTileThreads);
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_full[i], kTileThreads);
      mbar_init(&sh->item_full[i], 1);
      mbar_init(&sh->item_empty[i], kSoftmaxWarps);
      mbar_init(&sh->plan_full[2 * i], 1);
      mbar_init(&sh->plan_full[2 * i + 1], 1);
      mbar_init(&sh->plan_empty[2 * i], kLoadWarps);
      mbar_init(&sh->plan_empty[2 * i + 1], kLoadWarps);
      mbar_init(&sh->o_full[i], 1);
      mbar_init(&sh->described[i], 1);
    }
    mbar_init(&sh->drained, 1);
    fence_mbar_init();
  }
  if (warp == kThreads / 32 - 4) tmem_alloc(&sh->tmem, 512);
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // registers of the launch (896 x 72) shared out by role: 512 x 88 + 256 x 56 + 128 x 40
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    softmax_rows<T, D, Q8>(p, sh, q, warp >> 3, warp >> 2 & 1);
  } else if (warp < kSoftmaxWarps + kLoadWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    load_tiles<T, D, Q8>(p, sh, kv, reinterpret_cast<uint8_t *>(sh) + kHeader);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == kThreads / 32 - 3) plan_tiles<D>(p, sh);
    if (warp == kThreads / 32 - 4) issue_products<T, D, Q8>(p, sh, q, kv);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kThreads / 32 - 4) tmem_free(sh->tmem, 512);
}

}  // namespace

int launch_prefill(AttnParams &p, const yl_paged_attention_args *a, cudaStream_t stream) {
  auto go = [&](auto t, auto d, auto q8) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    constexpr bool Q8 = decltype(q8)::value;
    constexpr int smem = Shape<D>::kSmem + (Q8 ? Shape<D>::kRaw : 0);
    const int rc = allow_smem(reinterpret_cast<const void *>(prefill_kernel<T, D, Q8>), smem);
    if (rc != YL_OK) return rc;
    // no more items than full row tiles of the batch and one more per sequence
    const int64_t items = (a->num_tokens * p.group / Shape<D>::kRows + a->batch_size) * p.heads;
    return launch_dependent(prefill_kernel<T, D, Q8>, dim3(static_cast<unsigned>(std::min<int64_t>(items, sm_count()))),
                            dim3(kThreads), smem, stream, "yl_paged_attention launch", p);
  };
  auto kind = [&](auto t, auto d) {
    return a->kv_dtype == YL_KV_E4M3 ? go(t, d, std::true_type{}) : go(t, d, std::false_type{});
  };
  auto dim = [&](auto t) {
    if (a->head_dim == 64) return kind(t, std::integral_constant<int, 64>{});
    if (a->head_dim == 128) return kind(t, std::integral_constant<int, 128>{});
    return kind(t, std::integral_constant<int, 256>{});
  };
  return a->dtype == YL_DTYPE_BF16 ? dim(Bf16{}) : dim(Fp16{});
}

}  // namespace ylk
