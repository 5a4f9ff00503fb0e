// Attention of draft trees over the paged cache on the 5th-generation tensor
// cores (tcgen05 + TMEM), head_dim 128, fp16/bf16.
//
// Mathematics.  Row (node t, query head) of request r sees the committed keys
// max(ctx_start[first], ctx_start[t]) .. C - 1 and the drafted keys C + j
// whose ancestor bit j is set.  Softmax is the online form: a reference m, a
// sum l and an unnormalised O, each in fp32, so segments of the key axis
// merge exactly.
//
// What bounds it.  A tree of n nodes reads every committed K/V row once per
// KV head for n x G query rows: below about 240 rows (the machine's balance
// of bf16 operations and bytes) the time is the HBM read.
//
// Split.  An item is (request, KV head, up to two 128-row query tiles); its
// key axis is cut into 128-key tiles.  All tiles of all items lie on one cost
// axis (kTileCost per tile, kItemCost per item), of which each CTA takes an
// equal share, so the bytes are balanced whatever the lengths, and one long
// request spreads over the whole GPU.  Every CTA sums the costs itself from
// the metadata (a few KB): no planning launch, no host round trip.  An item
// cut by share borders leaves fp32 partials (at most a head and a tail per
// CTA), which the merge launch behind joins in a fixed order.
//
// Measured (B200, 6549 GB/s and 1624 bf16 TFLOP/s measured peaks, captured
// launches; fp16, then bf16 with its two products): 32 requests x 32 rows x
// 2.3K keys 72 us = 4235 GB/s and 76; 64 x 128 rows x 4K keys 209 us = 5123 GB/s
// and 245; 64 x 256 rows x 6K keys 479 us = 862 TFLOP/s and 602; 1 x 16 rows x
// 265 keys 17 and 18 us.  A call has a fixed part of about 17 us (8 until the
// first scores: metadata, block ids, first tiles; 9 for the last epilogue and
// the join).  In between, the HBM reads bound up to 128 rows of fp16.  What
// bounds two query tiles and bf16 is the chain scores, softmax, P.V of each
// stream, which two streams cover in part (P lies over S, so a stream's next
// scores wait for its P.V): per key tile of two query tiles 2048 cycles of MMA
// (3072 in bf16) and 2048 of exponentials.
//
// Inside a CTA (16 warps, roles without a block-wide barrier between items):
//   warp 11   scheduler: describes items in a 4-slot ring, loads their Q tiles
//   warps 8, 10  TMA producers of K (2 stages) and V (3 stages)
//   warp 9    MMA issuer
//   warps 0-3, 4-7  softmax of stream 0 and 1, one thread per row
//   warps 12-15  epilogue: joins, normalises and writes an item while the
//             softmax warps are in the next one
// The two streams each own S/P and O columns in TMEM.  With two query tiles
// (more than 128 rows) a stream is a query tile and both read every K/V tile.
// With one, both streams hold the same query tile and take the even and the
// odd key tiles: one stream's softmax runs under the other's MMAs, which a
// single tile could not overlap, and the streams' (m, l, O) merge in the
// epilogue.
//
// Rows of V that a query row does not see but another row does (other
// branches, window edges) may hold infinities or NaN, and 0 x NaN would reach
// O.  The V producer replaces the non-finite elements of those rows by 0 in
// shared memory; where it found any, the epilogue adds the seen ones back.
// Every mbarrier wait is bounded; a timeout sets kStatusWaitTimeout.
#include <math.h>

#include <mutex>
#include <type_traits>

#include "mvb_common.cuh"
#include "mvb_internal.h"
#include "ptx_sm100.cuh"

namespace mvb {
namespace {

using namespace sm100;

// sm100::mbar_wait with its loop kept a loop: unrolled at every call it made
// this kernel 160 KB of code, and each role's first steps of an item wait for
// instructions.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < (1 << 22); ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}

constexpr int kRows = 128;                 // MMA M: rows of one query tile
constexpr int kKeys = 128;                 // keys per KV tile
constexpr int kHalf = kRows * 128;         // [128 rows][64 elements] swizzled: 16 KiB
constexpr int kTileBytes = 2 * kHalf;      // [128][128] 16-bit
// A K/V tile: 8-row groups, each the swizzle atom of its columns 0-63 and then
// that of 64-127, so a page is one TMA box.
constexpr int kAtom = 1024, kGroupBytes = 2 * kAtom;
constexpr int kKStages = 2, kVStages = 3, kQStages = 2;
constexpr int kOffQ = 0;
constexpr int kOffK = kQStages * kTileBytes;
constexpr int kOffV = kOffK + kKStages * kTileBytes;
constexpr int kSmemBytes = kOffV + kVStages * kTileBytes;  // 224 KiB of the SM's 227
constexpr int kThreads = 512;
constexpr int kKProdWarp = 8, kMmaWarp = 9, kSchedWarp = 11;  // warp 10: V producer
constexpr int kEpiWarp = 12;                                  // warps 12-15: epilogue
constexpr int kItemSlots = 4;
constexpr int kItemReaders = 15;
constexpr int kFlagSlots = 8;  // items whose V flag may still be read (more than kItemSlots)
// Register split (setmaxnreg) of the launch's 512 x 128 between the two
// softmax warpgroups, the epilogue's and the one of the other roles.
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 168, kEpiRegs = 80, kOtherRegs = 96;
static_assert(2 * 128 * kSoftmaxRegs + 128 * kEpiRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs,
              "register split must fit the launch's registers");
constexpr uint32_t kTmemCols = 512;
__device__ __forceinline__ uint32_t col_s(int x) { return 128u * (uint32_t)x; }
__device__ __forceinline__ uint32_t col_o(int x) { return 256u + 128u * (uint32_t)x; }
// A row's reference moves to where its largest P is 2^kTop, once a P would pass
// 2^(kTop + kRescaleLog2).
constexpr float kRescaleLog2 = 8.f;

// Cost axis: a KV tile of an item with one or two query tiles, an item's
// fixed part, and the least share of a CTA.  Measured: kItemCost 12, 20 and 28
// give 81, 77 and 79 us at 32 x 32 rows x 2.3K keys (a regression of the CTAs'
// end times says 3 to 5 tiles an item); kMinShare 8 and 30 (2 or 7 tiles) give
// 17 and 20 us at 1 x 16 rows x 265 keys, where the GPU has room for the split.
constexpr int kTileCost1 = 4, kTileCost2 = 6, kItemCost = 20, kMinShare = 8;
static_assert(kMinShare >= kTileCost1 && kMinShare >= kTileCost2,
              "a share between an item's first and last holds a tile of it");

static_assert(drain_reaches_every_stage(kKStages) && drain_reaches_every_stage(kVStages) &&
                  drain_reaches_every_stage(kQStages),
              "an aborted CTA waits for every load it has in flight");

constexpr int kPartRows = 2 * kRows;  // rows of one partial

enum Bar : int {
  kQFull = 0,
  kQEmpty = kQFull + kQStages,
  kKFull = kQEmpty + kQStages,
  kKEmpty = kKFull + kKStages,
  kVFull = kKEmpty + kKStages,
  kVEmpty = kVFull + kVStages,
  kVReady = kVEmpty + kVStages,
  kSFull = kVReady + kVStages,   // +stream
  kPFull = kSFull + 2,           // +stream
  kPvDone = kPFull + 2,          // +stream
  kMl = kPvDone + 2,             // +stream: its (m, l) are in shared memory
  kORead = kMl + 2,              // the epilogue has read (m, l) and O of both streams
  kItemFull = kORead + 1,
  kItemEmpty = kItemFull + kItemSlots,
  kFinal = kItemEmpty + kItemSlots,
  kNumBars = kFinal + 1,
};

struct ItemDesc {
  int64_t q0, qe;       // first token of the item, end of the request's tokens
  int32_t r, h;         // request (-1: no more items), KV head
  int32_t n;            // KV tiles of this segment
  int32_t kbase;        // first key of the segment's first tile
  int32_t kv_lo, kv_hi; // keys any row may see: [kv_lo, kv_hi)
  int32_t committed;    // C: first drafted key
  int32_t lo_all;       // every row of the item sees committed keys from here
  int32_t two;          // two query tiles
  int32_t slot;         // partial slot, or -1: the whole item is this segment
  int32_t first, last;  // the segment holds the request's first / last tile
};

// What the merge needs of the item that a CTA starts and does not finish.
struct CutRecord {
  int64_t q0, qe, cost0;  // first token, end of tokens, place on the cost axis
  int64_t share;
  int32_t h, tiles, two, valid;
};

struct TreeParams {
  char* out;
  int32_t num_q_heads, num_kv_heads, group, block_q, block_size, bs_shift, box_rows, boxes;
  int64_t num_blocks, num_slots;
  const int64_t *qstart, *qsl, *ctx_len, *table;
  int64_t table_stride, table_width;
  const int64_t* mask;
  int32_t mask_words;
  int64_t num_tokens, num_requests;
  float scale_log2;
  float4* part_o;    // [CTA][2][32 column chunks][kPartRows]
  float2* part_ml;   // [CTA][2][kPartRows]
  CutRecord* cuts;   // [CTA]
  const char* cache;
  int32_t* status;
};

// Positions fit 32 bits (a context is at most 2^30 long).
__device__ __forceinline__ int32_t block_of(const TreeParams& p, int32_t pos) {
  return pos >> p.bs_shift;
}
__device__ __forceinline__ int32_t page_of(const TreeParams& p, const int64_t* trow, int32_t pos) {
  const int32_t lb = block_of(p, pos);
  if (lb >= p.table_width) return -1;
  const int64_t blk = __ldg(trow + lb);
  return (blk >= 0 && blk < p.num_blocks) ? (int32_t)blk : -1;
}
// Slot of position pos on page blk (slots of both planes fit 32 bits).
__device__ __forceinline__ int32_t slot_of(const TreeParams& p, int32_t blk, int32_t pos) {
  return (blk << p.bs_shift) + (pos & (p.block_size - 1));
}

__device__ __forceinline__ void touch(const int64_t* at) {
  [[maybe_unused]] int64_t v;
  asm volatile("ld.global.nc.b64 %0, [%1];\n" : "=l"(v) : "l"(at));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Bit 15 / 31 of the result: that 16-bit element's exponent is all ones.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t v) {
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  return ((v & 0x7fff7fffu) + (kBf16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}

// A request's place on the cost axis.
struct RequestCost {
  int32_t pairs, tiles, kbase;
  int64_t full, last, head;  // cost of an item with two query tiles, of the last item, of a KV head
};
__device__ __forceinline__ RequestCost cost_of(const TreeParams& p, const TreeExtent& e) {
  RequestCost c;
  const int32_t n = (int32_t)(e.qe - e.qs), two = 2 * p.block_q;
  c.pairs = (n + two - 1) / two;
  c.kbase = (int32_t)e.lo & ~(p.box_rows - 1);
  c.tiles = ((int32_t)e.hi - c.kbase + kKeys - 1) / kKeys;
  c.full = kItemCost + (int64_t)c.tiles * kTileCost2;
  const bool one = n - (c.pairs - 1) * two <= p.block_q;
  c.last = one ? kItemCost + (int64_t)c.tiles * kTileCost1 : c.full;
  c.head = (c.pairs - 1) * c.full + c.last;
  return c;
}
// First tile of an item at or behind cost position x (item at cost0).
__device__ __forceinline__ int32_t tile_at(int64_t x, int64_t cost0, bool two, int32_t tiles) {
  const int64_t d = x - cost0 - kItemCost;
  if (d <= 0) return 0;
  const int64_t j = two ? (d + kTileCost2 - 1) / kTileCost2 : (d + kTileCost1 - 1) / kTileCost1;
  return (int32_t)(j < tiles ? j : tiles);
}
template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attention_kernel(const __grid_constant__ CUtensorMap qmap,
                          const __grid_constant__ CUtensorMap kvmap, const TreeParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kNumBars];
  __shared__ __align__(16) ItemDesc items[kItemSlots];
  __shared__ float2 ml_sh[2][kRows];
  __shared__ int64_t warp_sum_sh[kThreads / 32];
  __shared__ int64_t start_prefix_sh;
  __shared__ int32_t start_request_sh;
  __shared__ int32_t bad_v_sh[kFlagSlots];
  __shared__ uint32_t tmem_base_sh;
  __shared__ int32_t abort_sh;
  __shared__ int32_t k_issued, v_issued, q_issued;  // TMA loads of tiles

  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int kParts = kBf16 ? 2 : 1;  // of P
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  allow_dependent_launch();  // the merge waits for this grid's end before it reads

  // ---- this CTA's share of the cost axis ----
  const int64_t per = (p.num_requests + kThreads - 1) / kThreads;
  const int64_t r_lo = min(tid * per, p.num_requests), r_hi = min(r_lo + per, p.num_requests);
  int64_t mine = 0;
#pragma unroll 1
  for (int64_t r = r_lo; r < r_hi; ++r) {
    TreeExtent e;
    if (tree_extent(p, r, e)) mine += cost_of(p, e).head * p.num_kv_heads;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) warp_sum_sh[warp] = incl;
  if (tid == 0) p.cuts[blockIdx.x].valid = 0;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int64_t v = warp_sum_sh[w];
    if (w < warp) before += v;
    total += v;
  }
  const int64_t share = max(axis_share(total, gridDim.x), (int64_t)kMinShare);
  const int64_t my_lo = blockIdx.x * share, my_hi = min(my_lo + share, total);
  if (my_lo >= total) return;
  if (before <= my_lo && my_lo < before + mine) {
    int64_t r = r_lo, at = before;
#pragma unroll 1
    for (;; ++r) {
      TreeExtent e;
      const int64_t c = tree_extent(p, r, e) ? cost_of(p, e).head * p.num_kv_heads : 0;
      if (my_lo < at + c) break;
      at += c;
    }
    start_request_sh = (int32_t)r;
    start_prefix_sh = at;
  }

  const uint32_t sb = smem_addr(smem);
  if ((sb & 1023u) != 0) {  // the swizzle needs the declared alignment
    if (tid == 0 && p.status != nullptr) atomicOr(p.status, kStatusWaitTimeout);
    return;
  }
  const uint32_t bar0 = smem_addr(&bars[0]);
  auto bar = [&](int i) { return bar0 + 8u * (uint32_t)i; };
  volatile int32_t* abort_flag = &abort_sh;

  if (tid == 0) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kvmap);
#pragma unroll 1
    for (int i = 0; i < kNumBars; ++i) {
      const bool four = (i >= kPFull && i < kPFull + 2) || (i >= kMl && i <= kORead) ||
                        (i >= kQEmpty && i < kQEmpty + kQStages);
      const bool readers = i >= kItemEmpty && i < kItemEmpty + kItemSlots;
      mbar_init(bar(i), readers ? kItemReaders : four ? 4 : 1);
    }
    mbar_init_fence();
    abort_sh = 0;
    k_issued = v_issued = q_issued = 0;
  }
  if (warp == kMmaWarp) tmem_alloc(smem_addr(&tmem_base_sh), kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;

  auto take_item = [&](uint32_t i, ItemDesc& d) -> bool {
    const uint32_t slot = i % kItemSlots;
    if (!__all_sync(0xffffffffu, bar_wait(bar(kItemFull + slot), (i / kItemSlots) & 1)))
      return false;
    d = items[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(kItemEmpty + slot));
    return true;
  };
  // KV tiles of stream x in an item of n tiles: all of them for a query tile
  // of its own, else every other one.
  auto stream_tiles = [](const ItemDesc& d, int x) { return d.two ? d.n : (d.n + 1 - x) >> 1; };
  // Running counts (identical in every role): KV tiles of this CTA, tiles per
  // stream, Q tiles.
  uint32_t kvc = 0, tc0 = 0, tc1 = 0, qc = 0;
  auto advance = [&](const ItemDesc& d) {
    kvc += (uint32_t)d.n;
    tc0 += (uint32_t)stream_tiles(d, 0);
    tc1 += (uint32_t)stream_tiles(d, 1);
    qc += d.two ? 2 : 1;
  };
  auto fail = [&]() {
    if (lane == 0) atomicOr(&abort_sh, 1);
  };
  auto kslot = [](uint32_t c) { return c % kKStages; };
  auto kphase = [](uint32_t c) { return (c / kKStages) & 1; };
  auto vslot = [](uint32_t c) { return c % kVStages; };
  auto vphase = [](uint32_t c) { return (c / kVStages) & 1; };

  // The row's keys among 32 from position k (row of token tok, window lo_q).
  auto seen32 = [&](const ItemDesc& d, int32_t lo_q, const uint64_t* mrow, uint64_t mask0,
                    int32_t k) -> uint32_t {
    const int32_t a = min(max(lo_q - k, 0), 32), b = min(max(d.committed - k, 0), 32);
    const uint32_t below_a = a >= 32 ? ~0u : (1u << a) - 1u, below_b = b >= 32 ? ~0u : (1u << b) - 1u;
    uint32_t bits = below_b & ~below_a;
    const int32_t j = k - d.committed, nodes = d.kv_hi - d.committed;  // first node of the 32
    if (j > -32 && j < nodes) {
      uint32_t tree;
      if (j <= 0) {
        tree = (uint32_t)(mask0 << (-j));
      } else {
        const int w = j >> 6, sh = j & 63;
        uint64_t v = (w == 0 ? mask0 : __ldg(mrow + w)) >> sh;
        if (sh > 32 && w + 1 < p.mask_words) v |= __ldg(mrow + w + 1) << (64 - sh);
        tree = (uint32_t)v;
      }
      if (nodes - j < 32) tree &= (1u << (nodes - j)) - 1u;
      bits |= tree;
    }
    return bits;
  };

  if (warp >= kEpiWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kEpiRegs));
    // ------------------------------------------------ epilogue
    // Joins the streams, normalises, and writes the item's rows or its
    // partial, while the softmax warpgroups are in the next item.  The loop
    // bodies are small: they run once per item, so fetching them counts.
    const int row = 32 * (warp & 3) + lane;  // TMEM lane of this thread
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    const int row_tok = row / p.group, row_head = row % p.group;
    for (uint32_t i = 0;; ++i) {
      ItemDesc d;
      if (!take_item(i, d)) {
        fail();
        break;
      }
      if (d.r < 0 || *abort_flag != 0) break;
      const int n0 = stream_tiles(d, 0), n1 = stream_tiles(d, 1);
      // A stream's last S is complete once its (m, l) are here, so its P.V
      // barrier is in the last tile's phase or just behind it.
      bool arrived = bar_wait(bar(kMl), i & 1) && bar_wait(bar(kMl + 1), i & 1) &&
                     bar_wait(bar(kPvDone), (tc0 + n0 - 1) & 1);
      if (n1 > 0) arrived = arrived && bar_wait(bar(kPvDone + 1), (tc1 + n1 - 1) & 1);
      if (!__all_sync(0xffffffffu, arrived)) {
        fail();
        break;
      }
      tc_fence_after();
      const bool bad = bad_v_sh[i % kFlagSlots] != 0;
      const float2 ml[2] = {ml_sh[0][row], ml_sh[1][row]};
      const int64_t part = (int64_t)blockIdx.x * 2 + d.slot;
      const int passes = d.two ? 2 : 1;
#pragma unroll 1
      for (int t = 0; t < passes; ++t) {  // query tiles
        const int64_t tok = d.q0 + (int64_t)t * p.block_q + row_tok;
        const bool row_valid = row < p.group * p.block_q && tok < d.qe;
        if (__any_sync(0xffffffffu, row_valid)) {
          float m_all = t == 0 ? ml[0].x : ml[1].x, l_all = t == 0 ? ml[0].y : ml[1].y;
          float f_a = 1.f, f_b = 0.f;
          const bool both = !d.two && n1 > 0;  // the row's other keys are in stream 1
          if (both) {
            m_all = fmaxf(ml[0].x, ml[1].x);
            const float mu = m_all == -INFINITY ? 0.f : m_all;
            f_a = ex2(ml[0].x - mu);
            f_b = ex2(ml[1].x - mu);
            l_all = ml[0].y * f_a + ml[1].y * f_b;
          }
          const float inv = l_all == 0.f ? 0.f : 1.f / l_all;
          const int part_row = t * kRows + row;
          if (d.slot >= 0 && row_valid) p.part_ml[part * kPartRows + part_row] = make_float2(m_all, l_all);
          // Every S of the item is done with its Q tile, which stages the output.
          uint8_t* qbuf = smem + kOffQ + (int)((qc + (uint32_t)t) % kQStages) * kTileBytes;
#pragma unroll 1
          for (int c0 = 0; c0 < 128; c0 += 16) {
            uint32_t o[16], u[16];
            tmem_ld16_raw(tmem + lane_base + col_o(t) + c0, o);
            if (both) tmem_ld16_raw(tmem + lane_base + col_o(1) + c0, u);
            tmem_wait_ld();
            reg_fence(o);
            reg_fence(u);
            float f[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              f[e] = __uint_as_float(o[e]) * f_a;
              if (both) f[e] = fmaf(__uint_as_float(u[e]), f_b, f[e]);
            }
            if (d.slot >= 0) {
              if (row_valid) {
                float4* dst = p.part_o + (part * 32 + c0 / 4) * kPartRows + part_row;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  dst[e * kPartRows] = make_float4(f[4 * e], f[4 * e + 1], f[4 * e + 2], f[4 * e + 3]);
              }
            } else {
              uint8_t* cell = qbuf + (c0 >> 6) * kHalf + row * 128;
#pragma unroll
              for (int e = 0; e < 2; ++e)
                *reinterpret_cast<uint4*>(cell + (((((c0 & 63) >> 3) + e) ^ (row & 7)) << 4)) =
                    make_uint4(pack2<T>(f[8 * e] * inv, f[8 * e + 1] * inv),
                               pack2<T>(f[8 * e + 2] * inv, f[8 * e + 3] * inv),
                               pack2<T>(f[8 * e + 4] * inv, f[8 * e + 5] * inv),
                               pack2<T>(f[8 * e + 6] * inv, f[8 * e + 7] * inv));
            }
            __syncwarp();
          }
        }
        if (bad && row_valid) {
          // The non-finite values that this row sees among the replaced ones,
          // added to what was just written.
          const int64_t* trow = p.table + (int64_t)d.r * p.table_stride;
          const uint64_t* mrow = reinterpret_cast<const uint64_t*>(p.mask) + tok * p.mask_words;
          const int32_t lo_q = (int32_t)min(max((int64_t)d.kv_lo, __ldg(p.qstart + tok)), (int64_t)d.committed);
          const int32_t seg_end = min(d.kbase + d.n * kKeys, d.kv_hi);
          uint8_t* qrow = smem + kOffQ + (int)((qc + (uint32_t)t) % kQStages) * kTileBytes + row * 128;
          float* prow = reinterpret_cast<float*>(p.part_o + part * 32 * kPartRows + t * kRows + row);
#pragma unroll 1
          for (int32_t k = max(d.kbase, d.kv_lo); k < seg_end; ++k) {
            if (k >= d.lo_all && k < d.committed) {
              k = d.committed - 1;
              continue;
            }
            if (!(seen32(d, lo_q, mrow, __ldg(mrow), k) & 1u)) continue;
            const int32_t blk = page_of(p, trow, k);
            if (blk < 0) continue;
            const T* v = reinterpret_cast<const T*>(p.cache) +
                         ((p.num_slots + slot_of(p, blk, k)) * p.num_kv_heads + d.h) * 128;
#pragma unroll 1
            for (int e = 0; e < 128; ++e) {
              const float f = to_float(v[e]);
              if (fabsf(f) < INFINITY) continue;
              if (d.slot >= 0) {
                prow[(e >> 2) * kPartRows * 4 + (e & 3)] += f;
              } else {
                T* cell = reinterpret_cast<T*>(qrow + (e >> 6) * kHalf +
                                               (((e & 63) >> 3) ^ (row & 7)) * 16) + (e & 7);
                *cell = from_float<T>(to_float(*cell) + f);
              }
            }
          }
        }
        __syncwarp();
        if (t == passes - 1) {  // O and (m, l) are read
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(kORead));
        }
      }
      if (d.slot < 0) {
        // Lane l stores 16-byte chunk l % 8 of row 4i + l / 8: whole lines.
#pragma unroll 1
        for (int t = 0; t < passes; ++t) {
          const int64_t tok = d.q0 + (int64_t)t * p.block_q + row_tok;
          const bool row_valid = row < p.group * p.block_q && tok < d.qe;
          const int64_t orow = tok * p.num_q_heads + (int64_t)d.h * p.group + row_head;
          const uint8_t* qbuf = smem + kOffQ + (int)((qc + (uint32_t)t) % kQStages) * kTileBytes;
          if (!__any_sync(0xffffffffu, row_valid)) continue;
#pragma unroll 2
          for (int it = 0; it < 16; ++it) {
            const int hf = it >> 3, r8 = 4 * (it & 7) + (lane >> 3);  // row of this warp
            const int64_t at = __shfl_sync(0xffffffffu, row_valid ? orow : -1, r8);
            const uint4 v = *reinterpret_cast<const uint4*>(
                qbuf + hf * kHalf + (row - lane + r8) * 128 + (((lane & 7) ^ (r8 & 7)) << 4));
            if (at >= 0)
              *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + at * 128 + 64 * hf + 8 * (lane & 7)) = v;
          }
        }
      }
      fence_proxy_async();  // the Q tiles may be loaded again
      __syncwarp();
      if (lane == 0)
        for (int t = 0; t < passes; ++t) mbar_arrive(bar(kQEmpty + (qc + (uint32_t)t) % kQStages));
      advance(d);
    }
  } else if (warp >= kKProdWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kOtherRegs));
    if (warp == kSchedWarp) {
      // ---------------------------------------------------- scheduler
      const uint32_t q_bytes = (uint32_t)(p.group * p.block_q) * 128u * 2u;
      int64_t r = start_request_sh, at = start_prefix_sh;  // request and its cost position
      int64_t batch = r;                                   // lane l holds request batch + l
      TreeExtent mine_e;
      bool mine_ok = batch + lane < p.num_requests && tree_extent(p, batch + lane, mine_e);
      int32_t h = 0, pair = 0;
      int64_t cost0 = at;  // of item (r, h, pair)
      bool fresh = true;   // the request's figures are not yet read
      TreeExtent e{};
      RequestCost rc{};
      CutRecord cut{};
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        // The next item with tiles in this share.
        ItemDesc d;
        d.r = -1;
#pragma unroll 1
        while (*abort_flag == 0) {
          if (fresh) {
            if (cost0 >= my_hi || r >= p.num_requests) break;
            if (r >= batch + 32) {
              batch = r;
              mine_ok = batch + lane < p.num_requests && tree_extent(p, batch + lane, mine_e);
            }
            const int src = (int)(r - batch);
            if (!__shfl_sync(0xffffffffu, mine_ok ? 1 : 0, src)) {
              ++r;
              continue;
            }
            e.qs = __shfl_sync(0xffffffffu, mine_e.qs, src);
            e.qe = __shfl_sync(0xffffffffu, mine_e.qe, src);
            e.lo = __shfl_sync(0xffffffffu, mine_e.lo, src);
            e.committed = __shfl_sync(0xffffffffu, mine_e.committed, src);
            e.hi = __shfl_sync(0xffffffffu, mine_e.hi, src);
            rc = cost_of(p, e);
            h = pair = 0;
            if (cost0 < my_lo) {  // the share begins inside this request
#pragma unroll 1
              for (; my_lo - cost0 >= rc.head; cost0 += rc.head) ++h;
#pragma unroll 1
              for (; pair < rc.pairs - 1 && my_lo - cost0 >= rc.full; cost0 += rc.full) ++pair;
            }
            fresh = false;
          }
          if (cost0 >= my_hi) break;
          const bool last_pair = pair == rc.pairs - 1;
          const int64_t cost = last_pair ? rc.last : rc.full;
          d.q0 = e.qs + (int64_t)pair * 2 * p.block_q;
          d.two = d.q0 + p.block_q < e.qe ? 1 : 0;
          const int32_t j0 = tile_at(my_lo, cost0, d.two, rc.tiles);
          const int32_t j1 = tile_at(my_hi, cost0, d.two, rc.tiles);
          const bool some = j1 > j0;
          if (some) {
            d.r = (int32_t)r;
            d.h = h;
            d.qe = e.qe;
            d.n = j1 - j0;
            d.kbase = rc.kbase + j0 * kKeys;
            d.kv_lo = (int32_t)e.lo;
            d.kv_hi = (int32_t)e.hi;
            d.committed = (int32_t)e.committed;
            d.first = j0 == 0;
            d.last = j1 == rc.tiles;
            d.slot = d.first && d.last ? -1 : d.first ? 1 : 0;
            if (d.first && !d.last) cut = {d.q0, e.qe, cost0, share, h, rc.tiles, d.two, 1};
          }
          cost0 += cost;
          if (!last_pair) {
            ++pair;
          } else {
            pair = 0;
            if (++h == p.num_kv_heads) {
              ++r;
              fresh = true;
            }
          }
          if (some) break;
        }
        if (d.r >= 0) {
          // Committed keys that every row of the item sees start here.
          int32_t hi_start = d.kv_lo;
          const int64_t tend = min(d.q0 + 2 * (int64_t)p.block_q, d.qe);
#pragma unroll 1
          for (int64_t t = d.q0 + lane; t < tend; t += 32)
            hi_start = max(hi_start, (int32_t)min(max(__ldg(p.qstart + t), (int64_t)0), (int64_t)d.committed));
#pragma unroll
          for (int o = 16; o > 0; o >>= 1)
            hi_start = max(hi_start, __shfl_xor_sync(0xffffffffu, hi_start, o));
          d.lo_all = hi_start;
        }
        const uint32_t slot = i % kItemSlots;
        if (!__all_sync(0xffffffffu,
                        bar_wait(bar(kItemEmpty + slot), ((i / kItemSlots) & 1) ^ 1))) {
          fail();
          break;
        }
        if (lane == 0) {
          items[slot] = d;
          mbar_arrive(bar(kItemFull + slot));
        }
        __syncwarp();
        if (d.r < 0) break;
        if (lane == 0) {
          const int qn = d.two ? 2 : 1;
#pragma unroll 1
          for (int t = 0; ok && t < qn; ++t) {
            const uint32_t c = qc + (uint32_t)t, qs = c % kQStages;
            if (!bar_wait(bar(kQEmpty + qs), ((c / kQStages) & 1) ^ 1)) {
              ok = false;
              break;
            }
            mbar_expect_tx(bar(kQFull + qs), q_bytes);
            const int32_t qy = d.h * p.group, qz = (int32_t)(d.q0 + (int64_t)t * p.block_q);
            tma_load_3d(sb + kOffQ + qs * kTileBytes, &qmap, 0, qy, qz, bar(kQFull + qs));
            tma_load_3d(sb + kOffQ + qs * kTileBytes + kHalf, &qmap, 64, qy, qz, bar(kQFull + qs));
            q_issued = (int32_t)c + 1;
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok) fail();
        // Under load a global load takes microseconds: bring what the other
        // warps read first of this item into the SM's cache.
#pragma unroll 1
        for (int64_t t = d.q0 + lane; t < min(d.q0 + 2 * (int64_t)p.block_q, d.qe); t += 32)
          touch(p.mask + t * p.mask_words);
        {
          const int32_t lb = block_of(p, d.kbase + max(d.n - 2, 0) * kKeys + 8 * lane);
          if (lb < p.table_width) touch(p.table + (int64_t)d.r * p.table_stride + lb);
        }
        advance(d);
      }
      if (lane == 0 && cut.valid) p.cuts[blockIdx.x] = cut;
    } else if (warp == kMmaWarp) {
      // ---------------------------------------------------- MMA issuer
      if (lane == 0) {
        const uint32_t idesc_qk = f16_idesc(kBf16, false, kRows, kKeys);
        const uint32_t idesc_pv = f16_idesc(kBf16, true, kRows, 128);
        const uint64_t dq0 = sw128_desc(sb + kOffQ, 16, 1024);
        const uint64_t dk0 = sw128_desc(sb + kOffK, 16, kGroupBytes);
        const uint64_t dv0 = sw128_desc(sb + kOffV, kAtom, kGroupBytes);
        auto s_step = [&](int x, uint32_t qs, uint32_t stage, int k) {
          const uint64_t dq = dq0 + (uint64_t)((qs * kTileBytes) >> 4);
          const uint64_t dk = dk0 + (uint64_t)((stage * kTileBytes) >> 4);
          const uint32_t q_step = (uint32_t)((k >> 2) * (kHalf >> 4) + 2 * (k & 3));
          const uint32_t k_step = (uint32_t)((k >> 2) * (kAtom >> 4) + 2 * (k & 3));
          umma_f16(tmem + col_s(x), dq + q_step, dk + k_step, idesc_qk, k > 0);
        };
        auto issue_s = [&](int x, uint32_t qs, uint32_t stage) {
#pragma unroll
          for (int k = 0; k < 8; ++k) s_step(x, qs, stage, k);
          umma_commit(bar(kSFull + x));
        };
        // An item's first S: rolled (measured: unrolled MMA issue in the tile
        // loops is 15 % of them, code fetched once per item costs more than it saves).
        auto issue_first_s = [&](int x, uint32_t qs, uint32_t stage) {
#pragma unroll 1
          for (int k = 0; k < 8; ++k) s_step(x, qs, stage, k);
          umma_commit(bar(kSFull + x));
        };
        // O_x += P_x . V of tile j.  16-key steps with no key of [kv_lo, kv_hi)
        // are left out: their V rows may hold anything.
        auto issue_pv = [&](const ItemDesc& d, int j, int x, uint32_t stage, bool acc) {
          const uint64_t dv = dv0 + (uint64_t)((stage * kTileBytes) >> 4);
          const uint32_t d_tmem = tmem + col_o(x), p_tmem = tmem + col_s(x);
          const int32_t k0 = d.kbase + (d.n - 1 - j) * kKeys;
          auto step = [&](int k, int part, bool add) {
            umma_f16_ts(d_tmem, p_tmem + 32 * (k >> 1) + 8 * (k & 1) + 16 * part,
                        dv + (uint64_t)(k * (2 * kGroupBytes >> 4)), idesc_pv, add);
          };
          if (k0 >= d.kv_lo && k0 + kKeys <= d.kv_hi) {
#pragma unroll
            for (int part = 0; part < kParts; ++part)
#pragma unroll
              for (int k = 0; k < 8; ++k) step(k, part, acc || k > 0 || part > 0);
          } else {
            const int lo = max(d.kv_lo - k0, 0) >> 4, hi = (min(d.kv_hi - k0, kKeys) + 15) >> 4;
#pragma unroll 1
            for (int k = lo; k < hi; ++k)
#pragma unroll
              for (int part = 0; part < kParts; ++part) step(k, part, acc || k > lo || part > 0);
          }
          umma_commit(bar(kPvDone + x));
        };
        // A probe costs ~200 cycles: V of tile c (landed and fixed) and, if
        // `more`, K tile ck go in one batch, while the MMAs issued before run.
        // V is waited for; k_ready says whether K is there.
        bool k_ready = true;
        auto wait_v = [&](uint32_t c, bool more, uint32_t ck) -> bool {
          const uint32_t vf = bar(kVFull + vslot(c)), vr = bar(kVReady + vslot(c));
          const uint32_t kf = more ? bar(kKFull + kslot(ck)) : vr;
          const uint32_t kp = more ? kphase(ck) : vphase(c);
          bool r0, r1;
          mbar_test3(vf, vphase(c), vr, vphase(c), kf, kp, r0, r1, k_ready);
          return (r0 || bar_wait(vf, vphase(c))) && (r1 || bar_wait(vr, vphase(c)));
        };
        auto wait_k = [&](uint32_t ck) -> bool {
          if (k_ready) return true;
          const bool there = bar_wait(bar(kKFull + kslot(ck)), kphase(ck));
          tc_fence_after();
          return there;
        };
        bool ok = true;
        for (uint32_t i = 0; ok; ++i) {
          const uint32_t slot = i % kItemSlots;
          if (!bar_wait(bar(kItemFull + slot), (i / kItemSlots) & 1)) {
            ok = false;
            break;
          }
          const ItemDesc d = items[slot];
          mbar_arrive(bar(kItemEmpty + slot));
          if (d.r < 0 || *abort_flag != 0) break;
          const int n = d.n;
          const uint32_t qs0 = qc % kQStages, qs1 = (qc + 1) % kQStages;
          ok = bar_wait(bar(kQFull + qs0), (qc / kQStages) & 1) &&
               bar_wait(bar(kKFull + kslot(kvc)), kphase(kvc));
          if (!ok) break;
          tc_fence_after();
          issue_first_s(0, qs0, kslot(kvc));
          if (!d.two) umma_commit(bar(kKEmpty + kslot(kvc)));
          if (d.two || n > 1) {  // stream 1: the other query tile, or the next KV tile
            const uint32_t c1 = kvc + (d.two ? 0 : 1);
            ok = d.two ? bar_wait(bar(kQFull + qs1), ((qc + 1) / kQStages) & 1)
                       : bar_wait(bar(kKFull + kslot(c1)), kphase(c1));
            if (!ok) break;
            tc_fence_after();
            issue_first_s(1, d.two ? qs1 : qs0, kslot(c1));
            umma_commit(bar(kKEmpty + kslot(c1)));
          }
          if (d.two) {
            ok = wait_v(kvc, n > 1, kvc + 1) && bar_wait(bar(kORead), (i & 1) ^ 1);
#pragma unroll 1
            for (int j = 0; ok && j < n; ++j) {
              const uint32_t c = kvc + j;
#pragma unroll 1
              for (int x = 0; x < 2; ++x) {
                ok = bar_wait(bar(kPFull + x), ((x == 0 ? tc0 : tc1) + j) & 1);
                if (!ok) break;
                tc_fence_after();
                issue_pv(d, j, x, vslot(c), j > 0);
                if (x == 1) umma_commit(bar(kVEmpty + vslot(c)));
                if (j + 1 < n) {
                  ok = x == 1 || wait_k(c + 1);
                  if (!ok) break;
                  issue_s(x, x == 0 ? qs0 : qs1, kslot(c + 1));
                  if (x == 1) {
                    umma_commit(bar(kKEmpty + kslot(c + 1)));
                    ok = wait_v(c + 1, j + 2 < n, c + 2);
                  }
                }
              }
            }
          } else {
            ok = wait_v(kvc, n > 2, kvc + 2) && bar_wait(bar(kORead), (i & 1) ^ 1);
#pragma unroll 1
            for (int j = 0; ok && j < n; ++j) {
              const uint32_t c = kvc + j;
              const int x = j & 1;
              ok = bar_wait(bar(kPFull + x), ((x == 0 ? tc0 : tc1) + (j >> 1)) & 1);
              if (!ok) break;
              tc_fence_after();
              issue_pv(d, j, x, vslot(c), j > 1);
              umma_commit(bar(kVEmpty + vslot(c)));
              if (j + 2 < n) {
                ok = wait_k(c + 2);
                if (!ok) break;
                issue_s(x, qs0, kslot(c + 2));
                umma_commit(bar(kKEmpty + kslot(c + 2)));
              }
              if (j + 1 < n) ok = wait_v(c + 1, j + 3 < n, c + 3);
            }
          }
          if (!ok) break;
          advance(d);
        }
        if (!ok) atomicOr(&abort_sh, 1);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------- producers
      const bool is_k = warp == kKProdWarp;
      // A V tile with rows that some query row does not see is fixed up once
      // it lands: rows behind the last key, before the first (within their
      // 16-key steps) and on missing pages are zeroed, the non-finite elements
      // of rows that only some query rows see too.  The fix waits in `todo`
      // while further loads can be sent.
      struct Todo {
        uint32_t c, item, boxes_ok;
        int32_t k0, kv_lo, kv_hi, lo_all, committed;
        bool last;
      } todo{};
      bool pending = false;
      uint32_t bad_v = 0;  // a non-finite element was replaced in the item
      auto leave_flag = [&](uint32_t item) {  // with the item's last tile
        const bool any = __any_sync(0xffffffffu, bad_v) != 0;
        if (lane == 0) bad_v_sh[item % kFlagSlots] = any ? 1 : 0;
        bad_v = 0;
      };
      auto fix_v = [&]() -> bool {
        pending = false;
        const uint32_t s = vslot(todo.c);
        if (!__all_sync(0xffffffffu, bar_wait(bar(kVFull + s), vphase(todo.c)))) return false;
        // Lane l takes 16-byte chunk l % 8 of row 4i + l / 8, both halves.
        uint8_t* vt = smem + kOffV + s * kTileBytes + (lane & 7) * 16;
        auto cell_of = [&](int row) {
          return reinterpret_cast<uint4*>(vt + (row >> 3) * kGroupBytes + (row & 7) * 128);
        };
        auto zero_rows = [&](int r0, int r1) {
#pragma unroll 1
          for (int row = r0 + (lane >> 3); row < r1; row += 4) {
            uint4* cell = cell_of(row);
            cell[0] = make_uint4(0, 0, 0, 0);
            cell[kAtom / 16] = make_uint4(0, 0, 0, 0);
          }
        };
        auto clean_rows = [&](int r0, int r1) {
#pragma unroll 1
          for (int row = r0 + (lane >> 3); row < r1; row += 4) {
            uint4* cell = cell_of(row);
            uint4 v[2] = {cell[0], cell[kAtom / 16]};
            uint32_t* w = reinterpret_cast<uint32_t*>(v);
            uint32_t any = 0;
#pragma unroll
            for (int q = 0; q < 8; ++q) any |= nonfinite2<T>(w[q]);
            if (any) {
              bad_v = 1;
#pragma unroll
              for (int q = 0; q < 8; ++q) w[q] &= ~((nonfinite2<T>(w[q]) >> 15) * 0xffffu);
              cell[0] = v[0];
              cell[kAtom / 16] = v[1];
            }
          }
        };
        const int lo = max(todo.kv_lo - todo.k0, 0), hi = min(todo.kv_hi - todo.k0, kKeys);
        zero_rows(lo & ~15, lo);  // 16-key steps beyond are not multiplied
        zero_rows(hi, (hi + 15) & ~15);
        if (todo.boxes_ok != (1u << p.boxes) - 1u)
#pragma unroll 1
          for (int b = 0; b < p.boxes; ++b)
            if (!((todo.boxes_ok >> b) & 1u)) zero_rows(b * p.box_rows, (b + 1) * p.box_rows);
        __syncwarp();
        clean_rows(lo, min(todo.lo_all - todo.k0, hi));
        clean_rows(max(todo.committed - todo.k0, lo), hi);
        fence_proxy_async();  // visible to the P.V MMAs
        if (todo.last) leave_flag(todo.item);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kVReady + s));
        return true;
      };
      bool ok = true;
      for (uint32_t i = 0; ok; ++i) {
        ItemDesc d;
        if (!take_item(i, d)) {
          ok = false;
          break;
        }
        const bool end = d.r < 0 || *abort_flag != 0;
        if (end && !pending) break;
        // Block ids of 32 boxes at a time, a group ahead: under load a lookup
        // takes longer than a tile.  Boxes count from the segment's first key;
        // group g holds the 32 that end 32 g before its last.
        const int n = end ? 1 : d.n;  // at the end, a fix may be left
        const int64_t* trow = p.table + (int64_t)max(d.r, 0) * p.table_stride;
        auto lookup = [&](int g) -> int32_t {
          const int b = n * p.boxes - 32 * (g + 1) + lane;
          return !end && b >= 0 ? page_of(p, trow, d.kbase + b * p.box_rows) : -1;
        };
        int32_t ids = -1, ids_next = lookup(0);
#pragma unroll 1
        for (int j = 0; ok && j < n; ++j) {
          const uint32_t c = kvc + j;
          const uint32_t s = is_k ? kslot(c) : vslot(c);
          const uint32_t full = bar((is_k ? kKFull : kVFull) + s);
          const uint32_t empty = bar((is_k ? kKEmpty : kVEmpty) + s);
          const uint32_t empty_phase = (is_k ? kphase(c) : vphase(c)) ^ 1;
          const int32_t k0 = d.kbase + (n - 1 - j) * kKeys;  // the drafted keys first
          const int32_t pos = k0 + p.box_rows * lane;
          const int in_group = (j * p.boxes) & 31;
          if (in_group == 0) {
            ids = ids_next;
            ids_next = lookup(j * p.boxes / 32 + 1);
          }
          const int32_t blk = __shfl_sync(0xffffffffu, ids, (32 - in_group - p.boxes + lane) & 31);
          const uint32_t boxes_ok = __ballot_sync(0xffffffffu, lane < p.boxes && blk >= 0);
          const bool last = j == n - 1;
          const bool dirty = k0 < d.lo_all || k0 + kKeys > d.committed ||
                             boxes_ok != (1u << p.boxes) - 1u;
          // A pending fix is done before the load when that has to wait, else
          // behind it: before the next fix, before the item's flag is left, or
          // when its tile is here.
#pragma unroll 1
          for (int step = 0; ok && step < 2; ++step) {
            bool fix = pending;
            if (step == 0) {
              fix = fix && (end || !__all_sync(0xffffffffu, mbar_test(empty, empty_phase)));
            } else {
              if (!__all_sync(0xffffffffu, bar_wait(empty, empty_phase))) {
                ok = false;
                break;
              }
              if (lane == 0) {
                (is_k ? k_issued : v_issued) = (int32_t)c + 1;
                mbar_expect_tx(full, kTileBytes);
              }
              __syncwarp();
              if (lane < p.boxes) {
                // Missing pages load page 0; the softmax masks their keys.
                const int32_t y = slot_of(p, max(blk, 0), pos) + (is_k ? 0 : (int32_t)p.num_slots);
                const uint32_t dst =
                    sb + (is_k ? kOffK : kOffV) + s * kTileBytes + lane * p.box_rows * 256;
                tma_load_4d(dst, &kvmap, 0, 0, 2 * d.h, y >> 3, full);
                if (is_k && blk < 0 && pos < d.kv_hi && pos + p.box_rows > d.kv_lo && p.status != nullptr)
                  atomicOr(p.status, MVB_STATUS_BLOCK_OUT_OF_RANGE);
              }
              fix = fix && (dirty || last ||
                            __all_sync(0xffffffffu, mbar_test(bar(kVFull + vslot(todo.c)), vphase(todo.c))));
            }
            if (fix) ok = fix_v();
            if (end) break;
          }
          if (is_k || end || !ok) continue;
          if (dirty) {
            todo = {c, i, boxes_ok, k0, d.kv_lo, d.kv_hi, d.lo_all, d.committed, last};
            pending = true;
          } else {
            if (last) leave_flag(i);
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kVReady + s));  // nothing to fix
          }
        }
        if (end) break;
        if (ok) advance(d);
      }
      if (!ok) fail();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------ softmax / epilogue of stream x
    const int x = warp >> 2;
    const int row = 32 * (warp & 3) + lane;  // TMEM lane of this thread
    const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t s_cols = tmem + lane_base + col_s(x);
    const uint32_t o_cols = tmem + lane_base + col_o(x);
    const int row_tok = row / p.group;
    for (uint32_t i = 0;; ++i) {
      ItemDesc d;
      if (!take_item(i, d)) {
        fail();
        break;
      }
      if (d.r < 0 || *abort_flag != 0) break;
      const int64_t* trow = p.table + (int64_t)d.r * p.table_stride;
      bool ok = true;
      const int qt = d.two ? x : 0;  // query tile of this stream
      const int64_t tok = d.q0 + (int64_t)qt * p.block_q + row_tok;
      const bool row_valid = row < p.group * p.block_q && tok < d.qe;
      const bool warp_valid = __any_sync(0xffffffffu, row_valid);
      const int32_t lo_q =
          row_valid ? (int32_t)min(max((int64_t)d.kv_lo, __ldg(p.qstart + tok)), (int64_t)d.committed) : 0;
      const uint64_t* mrow =
          reinterpret_cast<const uint64_t*>(p.mask) + (row_valid ? tok * p.mask_words : 0);
      const uint64_t mask0 = row_valid ? __ldg(mrow) : 0;  // in flight with the loads around it
      const int nx = stream_tiles(d, x), step = d.two ? 1 : 2, first = d.two ? 0 : x;
      const uint32_t tcx = x == 0 ? tc0 : tc1;
      float m_ref = -INFINITY, l = 0.f;
      int32_t blk_next = -1;
      if (lane < p.boxes && nx > 0)
        blk_next = page_of(p, trow, d.kbase + (d.n - 1 - first) * kKeys + p.box_rows * lane);
#pragma unroll 1
      for (int jj = 0; jj < nx; ++jj) {
        const int32_t k0 = d.kbase + (d.n - 1 - first - jj * step) * kKeys;
        const uint32_t pok = __ballot_sync(0xffffffffu, blk_next >= 0);
        blk_next = -1;
        if (lane < p.boxes && jj + 1 < nx)
          blk_next = page_of(p, trow, k0 - step * kKeys + p.box_rows * lane);
        const bool all_pages = pok == (1u << p.boxes) - 1u;
        // Does every row of this warp see every key of the tile?
        const bool whole = all_pages && k0 >= d.lo_all && k0 + kKeys <= d.committed;
        if (!__all_sync(0xffffffffu, bar_wait(bar(kSFull + x), (tcx + jj) & 1))) {
          ok = false;
          break;
        }
        tc_fence_after();
        if (warp_valid) {
          if (!whole) {
            // Scores of keys that the row does not see become -inf, in place
            // and in a small loop: one or two tiles of an item come here.
#pragma unroll 1
            for (int ch = 0; ch < 4; ++ch) {
              uint32_t seen = row_valid ? seen32(d, lo_q, mrow, mask0, k0 + 32 * ch) : 0u;
              if (!all_pages) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
                  if (!((pok >> ((32 * ch + 16 * u) / p.box_rows)) & 1u)) seen &= ~(0xffffu << (16 * u));
              }
              __syncwarp();
              uint32_t v[32];
              tmem_ld32_raw(s_cols + 32 * ch, v);
              tmem_wait_ld();
              reg_fence(v);
              float f[32];
#pragma unroll
              for (int e = 0; e < 32; ++e) f[e] = (seen >> e) & 1u ? __uint_as_float(v[e]) : -INFINITY;
              tmem_st32(s_cols + 32 * ch, f);
            }
            tmem_wait_st();
          }
          uint32_t sc[4][32];
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) tmem_ld32_raw(s_cols + 32 * ch, sc[ch]);
          tmem_wait_ld();
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) reg_fence(sc[ch]);
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < kKeys; e += 2)
            mx[(e >> 1) & 3] = fmax3(mx[(e >> 1) & 3], __uint_as_float(sc[e >> 5][e & 31]),
                                     __uint_as_float(sc[e >> 5][(e & 31) + 1]));
          // Rounded up, and compared by a difference: no P passes 2^(kTop + 8)
          // however large the scores are.
          const float tmax = __fmul_ru(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), p.scale_log2);
          // O / l is exact whatever the reference is.  fp16 holds [2^-14, 2^16)
          // in full: with P up to 2^15 a long tail of small weights comes
          // through (a weight is off by 2^-32 of the row's largest at most).
          // bf16 has fp32's exponents, and O less room for large values.
          constexpr float kTop = kBf16 ? 0.f : 7.f;
          float corr = 1.f;
          if (tmax - m_ref > kTop + kRescaleLog2) {  // (two infinities: no)
            const float m_new = tmax - kTop;
            corr = ex2(m_ref - m_new);  // 0 when m_ref is -inf
            l *= corr;
            m_ref = m_new;
          }
          // O holds P.V of the stream's tile before, complete because this S
          // (issued behind it) is.
          if (jj >= 1 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
            for (int ch = 0; ch < 8; ++ch) {
              uint32_t o[16];
              tmem_ld16_raw(o_cols + 16 * ch, o);
              tmem_wait_ld();
              reg_fence(o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st16(o_cols + 16 * ch, o);
            }
          }
          // P = 2^(s*scale - m), over S as packed 16-bit pairs (keys 32ch..+31
          // in columns 32ch..+15), summed before it is rounded.  A bf16 P goes
          // in two parts (the second in columns 32ch+16..+31) and two
          // products, as in the paged kernels: its first 8 bits, cut off, and
          // the rest rounded to 8 more.  2^-24 P on top keeps the rest above 0,
          // so that an infinity of V times it is no NaN.  With one part 64 x 128
          // rows x 4K keys take 199 us against 236, 3 x 244 rows x 48K 162
          // against 212.  The two parts' loop is rolled and reads its scores
          // from TMEM again, since code and registers count here: unrolled it
          // takes 330 instead of 270 us at 256 x 16 rows x 1K keys.
          const float mu = m_ref == -INFINITY ? 0.f : m_ref;
          const uint64_t scale2 = f32x2_pack(p.scale_log2, p.scale_log2);
          const uint64_t negmu2 = f32x2_pack(-mu, -mu);
          [[maybe_unused]] const uint64_t tiny2 = f32x2_pack(0x1p-24f, 0x1p-24f);
          uint64_t ps2[2] = {f32x2_pack(0.f, 0.f), f32x2_pack(0.f, 0.f)};
#pragma unroll(kBf16 ? 1 : 4)
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t again[32];
            if constexpr (kBf16) {
              __syncwarp();
              tmem_ld32_raw(s_cols + 32 * ch, again);
              tmem_wait_ld();
              reg_fence(again);
            }
            auto score = [&](int k) -> float {
              if constexpr (kBf16)
                return __uint_as_float(again[k]);
              else
                return __uint_as_float(sc[ch][k]);
            };
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              uint32_t pk[8], rest[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const int k = 16 * hh + 2 * e;
                float xa, xb;
                f32x2_unpack(f32x2_fma(f32x2_pack(score(k), score(k + 1)), scale2, negmu2), xa, xb);
                const float pa = ex2(xa), pb = ex2(xb);
                const uint64_t p2 = f32x2_pack(pa, pb);
                ps2[e & 1] = f32x2_add(ps2[e & 1], p2);
                if constexpr (kBf16) {
                  const uint32_t ua = __float_as_uint(pa), ub = __float_as_uint(pb);
                  pk[e] = __byte_perm(ua, ub, 0x7632);
                  const uint64_t first2 = f32x2_pack(__uint_as_float(ua & 0xffff0000u),
                                                     __uint_as_float(ub & 0xffff0000u));
                  float ra, rb;
                  f32x2_unpack(f32x2_fma(p2, tiny2, f32x2_sub(p2, first2)), ra, rb);
                  rest[e] = pack2<T>(ra, rb);
                } else {
                  pk[e] = pack2<T>(pa, pb);
                }
              }
              tmem_st8(s_cols + 32 * ch + 8 * hh, pk);
              if constexpr (kBf16) tmem_st8(s_cols + 32 * ch + 16 + 8 * hh, rest);
            }
          }
          tmem_wait_st();
          float s0, s1, s2, s3;
          f32x2_unpack(ps2[0], s0, s1);
          f32x2_unpack(ps2[1], s2, s3);
          l += (s0 + s1) + (s2 + s3);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kPFull + x));
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        fail();
        break;
      }

      // (m, l) go to the epilogue's warpgroup, which has read the item before.
      if (!__all_sync(0xffffffffu, bar_wait(bar(kORead), (i & 1) ^ 1))) {
        fail();
        break;
      }
      ml_sh[x][row] = make_float2(m_ref, l);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kMl + x));
      advance(d);
    }
  }

  // Everything this CTA issued lands before TMEM and shared memory go away.
  if (warp == kMmaWarp && lane == 0) {
    umma_commit(bar(kFinal));
    bar_wait(bar(kFinal), 0);
  }
  __syncthreads();
  if (abort_sh && tid == 0) {
    if (p.status != nullptr) atomicOr(p.status, kStatusWaitTimeout);
#pragma unroll 1
    for (int32_t c = first_in_flight(k_issued, kKStages); c < k_issued; ++c)
      bar_wait(bar(kKFull + kslot((uint32_t)c)), kphase((uint32_t)c));
#pragma unroll 1
    for (int32_t c = first_in_flight(v_issued, kVStages); c < v_issued; ++c)
      bar_wait(bar(kVFull + vslot((uint32_t)c)), vphase((uint32_t)c));
#pragma unroll 1
    for (int32_t c = first_in_flight(q_issued, kQStages); c < q_issued; ++c)
      bar_wait(bar(kQFull + c % kQStages), (c / kQStages) & 1);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
}

// Joins the partials of the items that were cut, and writes 0 to the rows that
// no request owns.  Every block finds the cut items itself; a job is 32 rows x
// 8 columns of one of them, a lane one row (the partials are column chunks of
// 4 with the rows adjacent: coalesced), and the jobs go round all warps of the
// grid, so that few items with many segments use the whole GPU too.  One block
// per SM: launching more costs more than the work.
constexpr int kMergeThreads = 1024;

template <typename T>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const TreeParams p, int32_t ctas) {
  __shared__ int32_t job_end[kMaxTreeCtas];  // jobs of cut items 0 .. i
  __shared__ int32_t warp_jobs[kMaxTreeCtas / 32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t warp0 = (int64_t)warp * gridDim.x + blockIdx.x;  // neighbours on different SMs
  const int64_t warps = (int64_t)gridDim.x * (kMergeThreads / 32);
  // The attention before does not write these rows, and its inputs were there
  // before it began.
  for_unowned_rows(p, lane, warp0, warps, [&](int64_t t0, int64_t t1) {
    const int64_t first = t0 * p.num_q_heads * 16, last = t1 * p.num_q_heads * 16;
    for (int64_t e = first + lane; e < last; e += 32)
      reinterpret_cast<uint4*>(p.out)[e] = make_uint4(0, 0, 0, 0);
  });
  grid_dependency_wait();
  if (tid < kMaxTreeCtas) {
    int32_t n = 0;
    if (tid < ctas && p.cuts[tid].valid) n = (p.cuts[tid].two ? 2 : 1) * (kRows / 32) * 16;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t u = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += u;
    }
    job_end[tid] = n;
    if (lane == 31) warp_jobs[warp] = n;
  }
  __syncthreads();
  if (tid < kMaxTreeCtas) {
    int32_t before = 0;
    for (int w = 0; w < warp; ++w) before += warp_jobs[w];
    job_end[tid] += before;
  }
  __syncthreads();
  const int32_t jobs = job_end[ctas - 1];
  for (int64_t job = warp0; job < jobs; job += warps) {
    int lo = 0, hi = ctas - 1;  // the first cut item that ends behind this job
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (job_end[mid] > job)
        hi = mid;
      else
        lo = mid + 1;
    }
    const int sub = (int)job - (lo > 0 ? job_end[lo - 1] : 0);
    const CutRecord c = p.cuts[lo];
    const int row = 32 * (sub >> 4) + lane;  // of the item's query tiles
    const int chunk = 2 * (sub & 15);
    const int in_tile = row & (kRows - 1);
    const int64_t tok = c.q0 + (int64_t)(row / kRows) * p.block_q + in_tile / p.group;
    if (in_tile >= p.group * p.block_q || tok >= c.qe) continue;
    // Every share from the item's first tile to its last holds some.
    const int b0 = lo;
    const int b_last = (int)divide(
        c.cost0 + kItemCost + (int64_t)(c.tiles - 1) * (c.two ? kTileCost2 : kTileCost1), c.share);
    float m = -INFINITY, l = 0.f;
    float o[8] = {};
#pragma unroll 4
    for (int b = b0; b <= b_last; ++b) {
      const int64_t part = 2 * b + (b == b0 ? 1 : 0);
      const float2 ml = __ldcg(p.part_ml + part * kPartRows + row);
      const float4 u = __ldcg(p.part_o + (part * 32 + chunk) * kPartRows + row);
      const float4 v = __ldcg(p.part_o + (part * 32 + chunk + 1) * kPartRows + row);
      const float m_new = fmaxf(m, ml.x), mu = m_new == -INFINITY ? 0.f : m_new;
      const float f0 = ex2(m - mu), f1 = ex2(ml.x - mu);
      m = m_new;
      l = l * f0 + ml.y * f1;
      const float add[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = o[e] * f0 + add[e] * f1;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t orow = tok * p.num_q_heads + (int64_t)c.h * p.group + in_tile % p.group;
    *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + orow * 128 + 4 * chunk) =
        make_uint4(pack2<T>(o[0] * inv, o[1] * inv), pack2<T>(o[2] * inv, o[3] * inv),
                   pack2<T>(o[4] * inv, o[5] * inv), pack2<T>(o[6] * inv, o[7] * inv));
  }
}

struct TreeDeviceState {
  bool checked = false, fits = false;
};
std::mutex g_tree_lock;
TreeDeviceState g_tree_state[kMaxDevices];

// The kernels were built with the register count that the split assumes, and
// take their shared memory on the current device.
bool tree_kernels_fit() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
  std::lock_guard<std::mutex> guard(g_tree_lock);
  TreeDeviceState& st = g_tree_state[dev];
  if (!st.checked) {
    const void* fns[2] = {reinterpret_cast<const void*>(tree_attention_kernel<__half>),
                          reinterpret_cast<const void*>(tree_attention_kernel<__nv_bfloat16>)};
    st.fits = true;
    for (const void* fn : fns) {
      cudaFuncAttributes fa;
      st.fits = st.fits && cudaFuncGetAttributes(&fa, fn) == cudaSuccess &&
                fa.maxThreadsPerBlock >= kThreads && fa.numRegs == kLaunchRegs &&
                cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes) == cudaSuccess;
    }
    st.checked = true;
  }
  return st.fits;
}

struct TreeLayout {
  size_t cuts, part_ml, part_o, end;
};
TreeLayout tree_layout(int64_t ctas) {
  TreeLayout w;
  auto align = [](size_t v) { return (v + 255) & ~(size_t)255; };
  w.cuts = 0;
  w.part_ml = align((size_t)ctas * sizeof(CutRecord));
  w.part_o = align(w.part_ml + (size_t)ctas * 2 * kPartRows * sizeof(float2));
  w.end = w.part_o + (size_t)ctas * 2 * 32 * kPartRows * sizeof(float4);
  return w;
}

// Rows of a TMA box: a page, or a tile's part of it.
int box_rows_of(int32_t block_size) { return block_size < kKeys ? block_size : kKeys; }

}  // namespace

size_t tree_workspace_bytes() { return tree_layout(kMaxTreeCtas).end; }

bool tree_tc_supported(const TreeProblem& a) {
  const int group = a.num_q_heads / a.num_kv_heads;
  const int64_t num_slots = a.num_blocks * a.block_size;
  return (a.dtype == MVB_DTYPE_F16 || a.dtype == MVB_DTYPE_BF16) && a.head_dim == 128 &&
         group <= 64 && a.block_size >= 16 && (a.block_size & (a.block_size - 1)) == 0 &&
         a.num_blocks > 0 &&
         ((uintptr_t)a.query % 16) == 0 && ((uintptr_t)a.cache % 16) == 0 &&
         ((uintptr_t)a.out % 16) == 0 &&
         (a.num_tokens == 1 || ((a.q_st % 8) == 0 && a.q_st >= 128)) &&
         (a.num_q_heads == 1 || ((a.q_sh % 8) == 0 && a.q_sh >= 128)) &&
         2 * num_slots < ((int64_t)1 << 31) && a.num_tokens < ((int64_t)1 << 31) &&
         a.num_requests < ((int64_t)1 << 31) && tensor_map_encoder() != nullptr && tree_kernels_fit();
}

int launch_tree_attention(const TreeProblem& a) {
  if (a.workspace == nullptr || ((uintptr_t)a.workspace % 256) != 0) return MVB_ERR_INVALID_ARGUMENT;
  const int ctas = num_sms() < kMaxTreeCtas ? num_sms() : kMaxTreeCtas;
  const TreeLayout w = tree_layout(ctas);
  if (a.workspace_bytes < w.end) return MVB_ERR_WORKSPACE_TOO_SMALL;
  EncodeTiled encode = tensor_map_encoder();
  const CUtensorMapDataType dt =
      a.dtype == MVB_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const int group = a.num_q_heads / a.num_kv_heads;
  const int64_t num_slots = a.num_blocks * a.block_size;
  const int box_rows = box_rows_of(a.block_size);
  CUtensorMap qmap, kvmap;
  {
    const cuuint64_t q_sh = a.num_q_heads == 1 ? 128 : (cuuint64_t)a.q_sh;
    const cuuint64_t q_st = a.num_tokens == 1 ? q_sh * a.num_q_heads : (cuuint64_t)a.q_st;
    const cuuint64_t dims[3] = {128, (cuuint64_t)a.num_q_heads, (cuuint64_t)a.num_tokens};
    const cuuint64_t strides[2] = {q_sh * 2, q_st * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)(kRows / group)};
    const cuuint32_t estr[3] = {1, 1, 1};
    if (encode(&qmap, dt, 3, const_cast<void*>(a.query), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return MVB_ERR_UNSUPPORTED_SHAPE;
  }
  {
    // [slot / 8][64-column segment][slot % 8][64 elements]: a box of a page is
    // 8-row groups of two segments, as the tiles lie in shared memory.
    const cuuint64_t row = (cuuint64_t)a.num_kv_heads * 256;
    const cuuint64_t dims[4] = {64, 8, (cuuint64_t)a.num_kv_heads * 2, (cuuint64_t)(2 * num_slots / 8)};
    const cuuint64_t strides[3] = {row, 128, 8 * row};
    const cuuint32_t box[4] = {64, 8, 2, (cuuint32_t)box_rows / 8};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    if (encode(&kvmap, dt, 4, const_cast<void*>(a.cache), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return MVB_ERR_UNSUPPORTED_SHAPE;
  }
  char* ws = static_cast<char*>(a.workspace);
  TreeParams p;
  p.out = static_cast<char*>(a.out);
  p.num_q_heads = a.num_q_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.group = group;
  p.block_q = kRows / group;
  p.block_size = a.block_size;
  p.bs_shift = __builtin_ctz(a.block_size);
  p.box_rows = box_rows;
  p.boxes = kKeys / box_rows;
  p.num_blocks = a.num_blocks;
  p.num_slots = num_slots;
  p.qstart = a.qstart;
  p.qsl = a.qsl;
  p.ctx_len = a.ctx_len;
  p.table = a.table;
  p.table_stride = a.table_stride;
  p.table_width = a.table_width;
  p.mask = a.mask;
  p.mask_words = a.mask_words;
  p.num_tokens = a.num_tokens;
  p.num_requests = a.num_requests;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.part_o = reinterpret_cast<float4*>(ws + w.part_o);
  p.part_ml = reinterpret_cast<float2*>(ws + w.part_ml);
  p.cuts = reinterpret_cast<CutRecord*>(ws + w.cuts);
  p.cache = static_cast<const char*>(a.cache);
  p.status = a.status;
  const bool bf16 = a.dtype == MVB_DTYPE_BF16;
  if (bf16)
    tree_attention_kernel<__nv_bfloat16><<<ctas, kThreads, kSmemBytes, a.stream>>>(qmap, kvmap, p);
  else
    tree_attention_kernel<__half><<<ctas, kThreads, kSmemBytes, a.stream>>>(qmap, kvmap, p);
  const int rc = check_launch();
  if (rc != MVB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = a.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = bf16 ? cudaLaunchKernelEx(&cfg, tree_merge_kernel<__nv_bfloat16>, p, ctas)
                             : cudaLaunchKernelEx(&cfg, tree_merge_kernel<__half>, p, ctas);
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return MVB_ERR_CUDA;
  }
  return check_launch();
}

}  // namespace mvb
