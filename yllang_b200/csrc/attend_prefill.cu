// Paged attention of sequences with many new tokens (prefill, chunks), for
// sm_100a: both products on the tensor cores, 4 * pairs * head_dim flops per
// query head.
//
// A work item is 2 x 128 query rows of one (sequence, KV head), a row being a
// (new token, head of the group), so a tile of keys serves the whole group.
// One CTA per SM walks items; its warps have fixed roles:
//
// * Warps 8-11 load: they gather rows of K and V by page, in tiles of KT tokens,
//   and leave them 16-bit and swizzled in a ring of two stages.  16-bit pools
//   are copied asynchronously; the codes of an 8-bit pool are converted on the
//   way to fp16, which holds every e4m3 value.  K's scales, relative to the
//   largest of the tile, are multiplied in (exact for powers of two); the tile's
//   largest goes to the scores as one factor.  V's are multiplied in relative to
//   a reference that changes only when a tile's largest passes 64 times it, when
//   the accumulators are rescaled.
// * Warp 12 (13 to 15 are there for the sharing out of registers) issues the products: S = Q K^T per 128 rows (both operands in shared
//   memory), O += P V (P in tensor memory).  The two row tiles alternate, so
//   that one's products run while the other's softmax does.
// * Warps 0-3 and 4-7 each own a row tile, one row per thread: they write Q into
//   shared memory (bf16 queries of an 8-bit pool become fp16 by a power of two
//   per row), then per tile of keys read S, keep the running maximum and sum in
//   fp32, and write the weights over S in 16 bits.  The maximum that the weights
//   refer to moves only when it grew by more than 2^8; then the row's
//   accumulator is rescaled.  fp16 weights are kept times 2^7, at most 2^15.
//
// Only tiles that some row does not see in full are masked; in those, infinities
// and NaN of V are zeroed as they are loaded and reported to the rows that see
// them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "attend_device.cuh"
#include "tcgen05.cuh"

namespace ylk {
namespace {

constexpr int kThreads = 16 * 32;
constexpr int kLoadThreads = 128;
constexpr int kStages = 2;
constexpr float kMoveBy = 8.f;    // log2 of how far weights may pass 1 before their reference moves
constexpr float kMaxRatio = 64.f; // of a V scale to the reference

template <int D>
struct Shape {
  static constexpr int kQTiles = D == 256 ? 1 : 2;  // 128-row tiles of an item
  static constexpr int kKT = D == 256 ? 64 : 128;   // tokens of a key tile
  static constexpr int kRows = 128 * kQTiles;
  static constexpr int kQBytes = 128 * D * 2;       // one row tile
  static constexpr int kKVBytes = kKT * D * 2;      // K or V of a stage
  static constexpr int kSmem = kQTiles * kQBytes + 2 * kStages * kKVBytes + 8192 + 1024;
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
  uint32_t valid[4]; // tokens with a good page
  uint32_t ghost[4]; // edge tiles: tokens whose V had an infinity or NaN
};

struct Shared {
  uint64_t k_full[kStages], v_full[kStages], k_empty[kStages], v_empty[kStages];
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t drained;
  uint32_t tmem;
  float top[2][2][4];           // [parity][K, V][loading warp]: largest scales
  uint32_t valid[2][4];         // [parity]: tokens with a good page
  TileInfo tile[kStages];
  int64_t offset[2][128];       // [parity]: byte offset of a token's head row
  uint32_t ratio[2][2][128];    // [parity][K, V]: scale over the reference, two halves
};
static_assert(sizeof(Shared) <= 8192, "shared header");

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
        out.first_pos = s.total - s.fresh + t0;
        out.last_pos = s.total - s.fresh + t1 - 1;
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
  if (mbar_wait_bounded(bar, parity, kBulkWaitLimitNs)) return true;
  raise_deverr(p.error_word, YL_DEVERR_TIMEOUT);
  return false;
}
// The same answer for the whole warp, which then goes on or leaves together.
__device__ __forceinline__ bool warp_wait(const AttnParams &p, uint64_t *bar, uint32_t parity) {
  const bool ok = mbar_wait_bounded(bar, parity, kBulkWaitLimitNs);
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
      "barrier.cta.red.and.pred p, 1, 128, q;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(all)
      : "r"(static_cast<uint32_t>(fine))
      : "memory");
  return all != 0;
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

// The tiles of this CTA's items, one after the other.
struct Tile {
  int base, cnt;            // first position and tokens of it
  int e0, head;             // of the sequence; KV head
  int first_pos, last_pos;  // of the item's queries
  bool first;               // of its item
};
template <int D>
class Tiles {
 public:
  __device__ __forceinline__ Tiles(const AttnParams &p) : walker_(p), n_(blockIdx.x) { more_ = walker_.seek(n_, it_); }
  // The next tile; false when there is none (cnt is 0 then).
  __device__ __forceinline__ bool next(Tile &t) {
    t.cnt = 0;
    if (!more_) return false;
    const bool in_head = j_ < it_.head_tiles;
    t.base = (in_head ? 0 : it_.span.low) + (in_head ? j_ : j_ - it_.head_tiles) * Shape<D>::kKT;
    t.cnt = min(Shape<D>::kKT, (in_head ? it_.span.head : it_.span.end) - t.base);
    t.e0 = it_.seq.e0;
    t.head = it_.head;
    t.first_pos = it_.first_pos;
    t.last_pos = it_.last_pos;
    t.first = j_ == 0;
    if (++j_ == it_.tiles) {
      j_ = 0;
      n_ += gridDim.x;
      more_ = walker_.seek(n_, it_);
    }
    return true;
  }

 private:
  Walker<D> walker_;
  Item it_;
  int64_t n_;
  int j_ = 0;
  bool more_;
};

// Each thread looks up one token of a tile: its page id two tiles ahead, the
// page's scales one tile ahead.
template <typename T, int D, bool Q8>
__device__ __forceinline__ void load_tiles(const AttnParams &p, Shared *sh, uint8_t *kv) {
  using S = Shape<D>;
  constexpr int KT = S::kKT;
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;
  constexpr int kNone = -0x7fffffff, kNoEntry = -0x7ffffffe;  // not a token of the tile; no such entry
  const int tid = threadIdx.x - 256, lane = tid & 31, warp = tid >> 5;
  Tiles<D> tiles(p);
  auto page_of = [&](const Tile &t) {
    if (tid >= KT || tid >= t.cnt) return kNone;
    const int64_t e = static_cast<int64_t>(t.e0) + p.by_page.div(t.base + tid);
    return e >= 0 && e < p.indices_cap ? __ldg(p.kv_indices + e) : kNoEntry;
  };
  auto good = [&](int page) { return page >= 0 && page < p.num_pages; };
  auto scales_of = [&](const Tile &t, int page, float &ks, float &vs) {
    ks = vs = 0.f;
    if (Q8 && good(page)) {
      const int64_t sc = static_cast<int64_t>(page) * p.scale_page_stride + t.head * p.scale_head_stride;
      ks = __ldg(p.scale[0] + sc);
      vs = __ldg(p.scale[1] + sc);
    }
  };
  Tile t0, t1, t2;
  bool more0 = tiles.next(t0), more1 = tiles.next(t1);
  int page0 = more0 ? page_of(t0) : kNone, page1 = more1 ? page_of(t1) : kNone;
  float ks0, vs0;
  scales_of(t0, page0, ks0, vs0);
  float value = 0.f;  // reference of V's scales
  for (uint32_t used = 0; more0; ++used) {
    const int stage = used % kStages, par = used & 1;
    const uint32_t phase = (used / kStages & 1) ^ 1;
    const bool more2 = tiles.next(t2);
    const int page2 = more2 ? page_of(t2) : kNone;
    float ks1 = 0.f, vs1 = 0.f;
    if (more1) scales_of(t1, page1, ks1, vs1);

    int64_t off = -1;
    if (good(page0)) {
      const int pos = t0.base + tid;
      off = static_cast<int64_t>(page0) * p.page_stride +
            static_cast<int64_t>(pos - static_cast<int>(p.by_page.div(pos)) * p.page_size) * p.slot_stride +
            t0.head * p.head_stride;
    } else if (page0 != kNone) {
      raise_deverr(p.error_word, page0 == kNoEntry ? YL_DEVERR_INDICES_CAP : YL_DEVERR_PAGE_RANGE);
    }
    if (tid < KT) sh->offset[par][tid] = off;
    const uint32_t ok = __ballot_sync(0xffffffffu, off >= 0);
    if (lane == 0 && warp * 32 < KT) sh->valid[par][warp] = ok;
    if (Q8) {
      float ktop = ks0, vtop = vs0;
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        ktop = fmaxf(ktop, __shfl_xor_sync(0xffffffffu, ktop, d));
        vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, d));
      }
      if (lane == 0) {
        sh->top[par][0][warp] = ktop;
        sh->top[par][1][warp] = vtop;
      }
    }
    load_barrier(true);
    float key = 1.f, move = 1.f;
    if (t0.first) value = Q8 ? 0.f : 1.f;
    if (Q8) {
      const float ktop = fmaxf(fmaxf(sh->top[par][0][0], sh->top[par][0][1]), fmaxf(sh->top[par][0][2], sh->top[par][0][3]));
      const float vtop = fmaxf(fmaxf(sh->top[par][1][0], sh->top[par][1][1]), fmaxf(sh->top[par][1][2], sh->top[par][1][3]));
      if (ktop > 0.f) key = ktop;
      if (vtop > value * kMaxRatio) {
        move = value / vtop;
        value = vtop;
      }
      if (tid < KT) {
        const float rk = ks0 / key, rv = value > 0.f ? vs0 / value : 0.f;
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
    constexpr int CH = D * (Q8 ? 1 : 2) / 16;    // 16-byte chunks of a token's head row
    constexpr int STEP = kLoadThreads / CH;      // rows of one pass of the threads
    constexpr int PER = KT / STEP;               // chunks of a thread
    const int c = tid % CH, r0 = tid / CH;
    uint4 w[Q8 ? PER : 1];
    if (Q8) {  // K's codes are on their way before the stage is free
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int64_t o = sh->offset[par][r0 + i * STEP];
        w[i] = make_uint4(0, 0, 0, 0);
        if (o >= 0) w[i] = __ldg(reinterpret_cast<const uint4 *>(p.kv[0] + o + c * 16));
      }
    }
    // the stage's previous tile is used up, its description too
    const bool fine = wait_or_report(p, &sh->k_empty[stage], phase) && wait_or_report(p, &sh->v_empty[stage], phase);
    TileInfo *info = &sh->tile[stage];
    if (tid == 0) {
      info->key = key;
      info->move = move;
      info->value = value;
      info->base = t0.base;
      info->edge = edge;
    }
    if (tid < KT / 32) {
      info->valid[tid] = sh->valid[par][tid];
      info->ghost[tid] = 0;
    }
    if (!load_barrier(fine)) break;

    if (Q8) {
      auto convert = [&](int i, int r, int kv_i) {
        const uint32_t ratio = sh->ratio[par][kv_i][r];
        const uint32_t x[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
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
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int r = r0 + i * STEP;
        convert(i, r, 0);
        const int64_t o = sh->offset[par][r];
        w[i] = make_uint4(0, 0, 0, 0);
        if (o >= 0) w[i] = __ldg(reinterpret_cast<const uint4 *>(p.kv[1] + o + c * 16));
      }
      fence_to_async();
      mbar_arrive(&sh->k_full[stage]);
#pragma unroll
      for (int i = 0; i < PER; ++i) convert(i, r0 + i * STEP, 1);
      fence_to_async();
      mbar_arrive(&sh->v_full[stage]);
    } else {
#pragma unroll
      for (int kv_i = 0; kv_i < 2; ++kv_i) {
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
    t0 = t1;
    t1 = t2;
    more0 = more1;
    more1 = more2;
    page0 = page1;
    page1 = page2;
    ks0 = ks1;
    vs0 = vs1;
  }
  cp_async_wait_all();
}

// ---------------------------------------------------------------------------
// Product warp (one thread)
// ---------------------------------------------------------------------------
template <typename T, int D, bool Q8>
__device__ __forceinline__ void issue_products(const AttnParams &p, Shared *sh, uint8_t *q, uint8_t *kv) {
  using S = Shape<D>;
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;
  constexpr int KT = S::kKT;
  constexpr uint32_t kScores = f16_product(BF, 128, KT, false), kValues = f16_product(BF, 128, D, true);
  const int lane = threadIdx.x & 31;
  const uint32_t tmem = sh->tmem, sq = smem_addr(q), skv = smem_addr(kv);
  Walker<D> walker(p);
  Item it;
  uint32_t used = 0;
  uint32_t queries[2] = {0, 0}, weights[2] = {0, 0};  // waits on q_full and p_full so far
  bool ok = true;
  for (int64_t n = blockIdx.x; walker.seek(n, it); n += gridDim.x) {
    const int live = min(S::kQTiles, (it.rows - it.row0 + 127) / 128);
    if (lane == 0 && ok) {
      auto scores = [&](int w, uint32_t tile) {
        const uint32_t a = sq + w * S::kQBytes, b = skv + (tile % kStages) * 2 * S::kKVBytes;
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
          mma_ss(tmem + S::kS + w * KT, tile_desc(a + (s / 4) * (128 * 128) + (s % 4) * 32, 16),
                 tile_desc(b + (s / 4) * (KT * 128) + (s % 4) * 32, 16), kScores, s > 0);
        mma_commit(&sh->s_full[w]);
        if (w == live - 1) mma_commit(&sh->k_empty[tile % kStages]);
      };
      ok = wait_or_report(p, &sh->k_full[used % kStages], used / kStages & 1);
      fence_to_async();  // (asynchronous copies of a 16-bit pool arrive without one)
      for (int w = 0; w < live && ok; ++w) {
        ok = wait_or_report(p, &sh->q_full[w], queries[w]++ & 1);
        if (!ok) break;
        tc_fence_after();
        scores(w, used);
      }
      for (int j = 0; j < it.tiles && ok; ++j) {
        const uint32_t tile = used + j;
        ok = wait_or_report(p, &sh->v_full[tile % kStages], tile / kStages & 1);
        fence_to_async();
        for (int w = 0; w < live && ok; ++w) {
          ok = wait_or_report(p, &sh->p_full[w], weights[w]++ & 1);
          if (!ok) break;
          tc_fence_after();
          const uint32_t b = skv + (tile % kStages) * 2 * S::kKVBytes + S::kKVBytes;
#pragma unroll
          for (int s = 0; s < KT / 16; ++s)
            mma_ts(tmem + S::kO + w * D, tmem + S::kS + w * KT + s * 8, tile_desc(b + s * 2048, KT * 128), kValues,
                   j > 0 || s > 0);
          if (w == live - 1) mma_commit(&sh->v_empty[tile % kStages]);
          if (j + 1 < it.tiles) {
            if (w == 0) {
              ok = wait_or_report(p, &sh->k_full[(tile + 1) % kStages], (tile + 1) / kStages & 1);
              if (!ok) break;
              fence_to_async();
            }
            scores(w, tile + 1);
          } else {
            mma_commit(&sh->o_full[w]);
          }
        }
      }
    }
    used += it.tiles;
    __syncwarp();
  }
  if (lane == 0) {
    // nothing of this CTA is in flight when its tensor memory goes
    mma_commit(&sh->drained);
    wait_or_report(p, &sh->drained, 0);
  }
  __syncwarp();
}

// ---------------------------------------------------------------------------
// Softmax warps: row tile w, one row per thread
// ---------------------------------------------------------------------------
// The lowest n bits, n of any sign.
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}

// This row's accumulator times a factor (rare: the reference of the weights moved).
template <int D>
__device__ __forceinline__ void rescale(uint32_t at, float factor) {
#pragma unroll 1
  for (int k = 0; k < D / 32; ++k) {
    uint32_t x[32];
    tmem_ld32(at + 32 * k, x);
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * factor);
    tmem_st32(at + 32 * k, x);
  }
}

template <typename T, int D, bool Q8>
__device__ __forceinline__ void softmax_rows(const AttnParams &p, Shared *sh, uint8_t *q, int w) {
  using S = Shape<D>;
  constexpr int KT = S::kKT;
  constexpr bool BF = std::is_same<T, Bf16>::value && !Q8;
  constexpr float kLift = BF ? 0.f : 7.f;
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
  const int r = warp * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
  const uint32_t ts = sh->tmem + lanes + S::kS + w * KT, to = sh->tmem + lanes + S::kO + w * D;
  const uint32_t sq = smem_addr(q) + w * S::kQBytes;
  Walker<D> walker(p);
  Item it;
  uint32_t used = 0, waits = 0, done = 0;
  for (int64_t n = blockIdx.x; walker.seek(n, it); n += gridDim.x) {
    if (w >= S::kQTiles || it.row0 + w * 128 >= it.rows) {  // an item without this row tile
      used += it.tiles;
      continue;
    }
    const int row = it.row0 + w * 128 + r;
    const int t = p.by_group.div(min(row, it.rows - 1)), g = min(row, it.rows - 1) - t * p.group;
    const int64_t qrow = static_cast<int64_t>(it.seq.q0) + t;
    const bool has = row < it.rows && qrow < p.num_tokens;
    const int pos = it.seq.total - it.seq.fresh + t;
    const int64_t h = static_cast<int64_t>(it.head) * p.group + g;

    // this row's query, 16-bit and swizzled
    float coef = p.scale_log2;
    {
      const uint4 *src = reinterpret_cast<const uint4 *>(p.q + (has ? qrow * p.q_row_stride + h * p.q_head_stride : 0));
      float up = 1.f;
      if (Q8 && std::is_same<T, Bf16>::value) {
        uint32_t big = 0;
#pragma unroll 8
        for (int c = 0; c < D / 8; ++c) {
          const uint4 x = has ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
          big = __vmaxu2(big, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                       __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
        }
        big = max(big & 0xffffu, big >> 16);
        const int e = min(max(static_cast<int>(big >> 7), 1), 253);  // biased exponent of the largest element
        up = __uint_as_float(static_cast<uint32_t>(254 - e) << 23);
        coef *= __uint_as_float(static_cast<uint32_t>(e) << 23);
      }
#pragma unroll 8
      for (int c = 0; c < D / 8; ++c) {
        uint4 x = has ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
        if (Q8 && std::is_same<T, Bf16>::value) {
          auto turn = [&](uint32_t &v) {
            const float2 f = Bf16::unpack(v);
            v = Fp16::pack(f.x * up, f.y * up);
          };
          turn(x.x);
          turn(x.y);
          turn(x.z);
          turn(x.w);
        }
        sts128(sq + swizzled<128>(r, c), x.x, x.y, x.z, x.w);
      }
      fence_to_async();
      tc_fence_before();  // the previous item's accumulators are read
      mbar_arrive(&sh->q_full[w]);
    }

    float m = -INFINITY, l = 0.f, value = 1.f;
    for (int j = 0; j < it.tiles; ++j, ++used) {
      const int stage = used % kStages;
      const uint32_t phase = used / kStages & 1;
      if (!warp_wait(p, &sh->s_full[w], waits++ & 1)) return;
      if (!warp_wait(p, &sh->k_full[stage], phase)) return;  // (over: the description is the loading warps')
      tc_fence_after();
      const TileInfo *info = &sh->tile[stage];
      const float c = coef * info->key;
      const float move = info->move;
      const bool edge = info->edge != 0;
      value = info->value;
      if (edge && !warp_wait(p, &sh->v_full[stage], phase)) return;  // which values were no numbers
      // The scores in chunks of 64 columns: the maximum over all, the last chunk
      // first; then the weights, the first chunk first (it is still in registers),
      // each written over scores that are used up.
      uint32_t x[64];
      auto load = [&](int h) {
        tmem_ld64(ts + 64 * h, x);
        if (edge) {
          // columns that this row sees: up to `last`, and past `out` or before `sink`
          const int base = info->base + 64 * h;
          const int last = pos - base + 1, out = p.window > 0 ? pos - p.window - base + 1 : 0;
          const int sink = p.window > 0 ? p.sinks - base : 0;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t see =
                info->valid[2 * h + k] & low_bits(last - 32 * k) & (~low_bits(out - 32 * k) | low_bits(sink - 32 * k));
            const uint32_t ghost = info->ghost[2 * h + k] & see;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((see >> i) & 1u)) x[32 * k + i] = 0xff800000u;  // -inf
            if (ghost) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if ((ghost >> i) & 1u) x[32 * k + i] = 0x7fffffffu;  // NaN
            }
          }
        }
      };
      float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int h = KT / 64 - 1; h >= 0; --h) {
        load(h);
#pragma unroll
        for (int i = 0; i < 64; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            tops[k] = fmaxf(tops[k], fmaxf(__uint_as_float(x[i + 2 * k]), __uint_as_float(x[i + 2 * k + 1])));
      }
      const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * c;
      float factor = move;
      if (top > m + kMoveBy) {
        const float f = fast_exp2(m - top);
        m = top;
        l *= f;
        factor *= f;
      }
      const bool moved = j > 0 && __any_sync(0xffffffffu, factor != 1.f);
      const float off = kLift - (m == -INFINITY ? 0.f : m);
      float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int h = 0; h < KT / 64; ++h) {
        if (h > 0) load(h);
        uint32_t y[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float a = fast_exp2(fmaf(__uint_as_float(x[2 * i]), c, off));
          const float b = fast_exp2(fmaf(__uint_as_float(x[2 * i + 1]), c, off));
          sums[2 * (i & 1)] += a;
          sums[2 * (i & 1) + 1] += b;
          y[i] = BF ? Bf16::pack(a, b) : Fp16::pack(a, b);
        }
        tmem_st32(ts + 32 * h, y);
      }
      if (moved) rescale<D>(to, factor);
      l += (sums[0] + sums[1]) + (sums[2] + sums[3]);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&sh->p_full[w]);
    }

    if (!warp_wait(p, &sh->o_full[w], done++ & 1)) return;
    tc_fence_after();
    const float inv = l == 0.f ? 0.f : value / l;
    char *out = p.o + (has ? qrow * p.o_row_stride + h * p.o_head_stride : 0);
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      uint32_t x[32];
      tmem_ld32(to + 32 * k, x);
      if (has) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          uint32_t y[4];
#pragma unroll
          for (int a = 0; a < 4; ++a)
            y[a] = T::pack(__uint_as_float(x[i + 2 * a]) * inv, __uint_as_float(x[i + 2 * a + 1]) * inv);
          *reinterpret_cast<uint4 *>(out + (32 * k + i) * 2) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
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
      mbar_init(&sh->q_full[i], 128);
      mbar_init(&sh->s_full[i], 1);
      mbar_init(&sh->p_full[i], 128);
      mbar_init(&sh->o_full[i], 1);
    }
    mbar_init(&sh->drained, 1);
    fence_mbar_init();
  }
  if (warp == 12) tmem_alloc(&sh->tmem, 512);
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // registers of the launch (512 x 128) shared out by role: 256 x 152 + 128 x 112 + 128 x 96
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    softmax_rows<T, D, Q8>(p, sh, q, warp >> 2);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 112;");
    load_tiles<T, D, Q8>(p, sh, kv);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 12) issue_products<T, D, Q8>(p, sh, q, kv);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 12) tmem_free(sh->tmem, 512);
}

}  // namespace

int launch_prefill(AttnParams &p, const yl_paged_attention_args *a, cudaStream_t stream) {
  auto go = [&](auto t, auto d, auto q8) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    constexpr bool Q8 = decltype(q8)::value;
    const int rc = allow_smem(reinterpret_cast<const void *>(prefill_kernel<T, D, Q8>), Shape<D>::kSmem);
    if (rc != YL_OK) return rc;
    // no more items than full row tiles of the batch and one more per sequence
    const int64_t items = (a->num_tokens * p.group / Shape<D>::kRows + a->batch_size) * p.heads;
    return launch_dependent(prefill_kernel<T, D, Q8>, dim3(static_cast<unsigned>(std::min<int64_t>(items, sm_count()))),
                            dim3(kThreads), Shape<D>::kSmem, stream, "yl_paged_attention launch", p);
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
