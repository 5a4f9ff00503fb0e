// Attention of draft trees over the paged cache for every shape that the
// tcgen05 kernel does not take: fp32, any head_dim up to 256, any block size,
// any GQA ratio.
//
// A CTA takes 32 query rows (node, head of one GQA group) of a request and KV
// head, and walks the request's keys in tiles of 64: K and V rows come into
// shared memory once for the 32 rows, as fp32.  q.k and P.V run on the tensor
// cores (mma.sync, TF32 operands, fp32 sums) with fp32 accuracy: a value is
// hi + lo (21 bits of it count), a product hi hi + hi lo + lo hi.  fp16 and
// bf16 values have no lo.  The tensor cores cut off what a sum cannot hold, half
// a last bit each time on average, so the hi products go round several sums (4
// for q.k, 2 for P.V) and the small ones have their own: one sum for all was
// 1.4e-6 off at 24 x 1.5K keys, against 5e-7 of a plain fp32 product; this is
// 2.4e-7 off and costs 3 % (200 x 128 x 1K keys 2.97 -> 3.06 ms, 64 x 32 x 1.5K
// 350 -> 362 us).
// The softmax is fp32, a warp owning 4 rows, their statistics in registers.
// Tiles that hold infinities or NaN go through scalar loops: hi and lo of an
// infinity are no sum, and what a row does not see must not reach it as 0 x NaN.
//
// Measured (B200, fp32, captured launches): 5 requests x 48 rows x up to 1.5K
// keys 39 us, 64 x 32 x 1.5K keys 362 us and 200 x 128 x 1K keys 3.06 ms (34
// TFLOP/s of useful products), 1 x 128 x 8K keys 129 us, 1 x 16 x 64 keys 15 us.
// A tile takes a CTA 14K cycles beside the SM's other CTA: a third q.k, a third
// P.V, a sixth the copies' instructions, a twelfth each the softmax and the
// checks for infinities.  The tensor pipe is active for 40 % of the time and 55 %
// of the cycles issue (2114 instructions per warp and tile, 192 of them tensor:
// fragments are loaded as single words, and K and V cut into hi and lo by each
// warp that reads them), with 16 warps an SM to cover latencies.  K and V rows
// by bulk copies of one warp instead of cp.async by all took 516 against 369 us
// at 64 x 32 x 1.5K keys.  On the CUDA cores the same tiles are bound by shared
// memory (12-18 TFLOP/s; two operand loads for 32 FMA instructions).
//
// Split.  An item is (32 query rows, KV head); the key tiles of all items lie
// on one axis with kItemCost for each item's fixed part, and every CTA takes an
// equal share of it, which it finds itself from the metadata.  An item that
// share borders cut leaves (max, sum, weighted V) partials, at most a head and a
// tail per CTA, which the join launch behind adds up in order.
#include <math.h>

#include <mutex>
#include <type_traits>

#include "mvb_common.cuh"
#include "mvb_internal.h"

namespace mvb {
namespace {

constexpr int kThreads = 256;
constexpr int kRowTile = 32, kWarpRows = 4;
constexpr int kKeyTile = 64;
constexpr int kMaxCtas = 2 * kMaxTreeCtas;
// In key tiles.  1, 2 and 4 give 89, 96 and 96 us at 5 x 48 rows x 2K keys, and
// 369, 368 and 385 us at 64 x 32 x 1.5K.
constexpr int kItemCost = 1;

// What the join needs of the item that a CTA starts and does not finish.
struct CutItem {
  int64_t qs, cost0, share;  // the request's first token; the item's place on the axis
  int32_t row0, n_rows, h, tiles, valid;
};

struct GenericParams {
  float scale_log2;
  float* part_o;    // [CTA][2][kRowTile][head_dim]
  float2* part_ml;  // [CTA][2][kRowTile] (max, sum)
  CutItem* cuts;    // [CTA]
};

// A request's place on the cost axis.
struct RequestItems {
  int32_t n_rows, row_tiles, tiles, items;
  int64_t cost;  // of an item
};
__device__ __forceinline__ RequestItems items_of(const TreeProblem& p, const TreeExtent& e, int32_t group) {
  RequestItems q;
  q.n_rows = (int32_t)(e.qe - e.qs) * group;
  q.row_tiles = (q.n_rows + kRowTile - 1) / kRowTile;
  q.tiles = ((int32_t)(e.hi - e.lo) + kKeyTile - 1) / kKeyTile;
  q.items = q.row_tiles * p.num_kv_heads;
  q.cost = kItemCost + q.tiles;
  return q;
}

template <typename T>
__device__ __forceinline__ float4 load4(const T* at);
template <>
__device__ __forceinline__ float4 load4<__half>(const __half* at) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16* at) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(at));
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// x = hi + lo, hi rounded to TF32 (10 mantissa bits; in integers, since
// conversions run at a quarter of the rate).  The tensor cores take the upper
// 19 bits of lo, so 21 bits of x count.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// 16 bytes to shared memory, zeros where `there` is false (src is not read).
__device__ __forceinline__ void copy16(float* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(
                   (uint32_t)__cvta_generic_to_shared(dst)),
               "l"(src), "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
__device__ __forceinline__ void copy_wait_but_last() {
  asm volatile("cp.async.wait_group 1;\n" ::: "memory");
}

// NT: 8-column tiles of a warp (head_dim <= 32 NT).  kVec: cache rows are
// whole, aligned 4-element vectors.
template <typename T, int NT, bool kVec>
__global__ void __launch_bounds__(kThreads, NT <= 4 ? 2 : 1)
    tree_attention_generic_kernel(const TreeProblem p, const GenericParams g) {
  constexpr int kDim = 32 * NT;                            // padded columns (zeros behind head_dim)
  constexpr int kQStride = kDim + 4, kVStride = kDim + 8;  // conflict-free fragment loads
  constexpr int kKStride = kDim + 4;
  constexpr int kSStride = kKeyTile + 4;
  constexpr bool kFp32 = std::is_same<T, float>::value;    // q, k and v have a lo
  constexpr int kQParts = kFp32 ? 2 : 1;
  extern __shared__ __align__(16) float sm[];
  __shared__ int64_t warp_sum_sh[kThreads / 32];
  __shared__ int64_t start_r_sh, start_at_sh;
  __shared__ int64_t slots_sh[2][kKeyTile];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t dim = p.head_dim, group = p.num_q_heads / p.num_kv_heads;
  T* out = static_cast<T*>(p.out);
  allow_dependent_launch();  // the join waits for this grid's end before it reads

  // This CTA's share of the cost axis.
  const int64_t per = (p.num_requests + kThreads - 1) / kThreads;
  const int64_t r_lo = min(tid * per, p.num_requests), r_hi = min(r_lo + per, p.num_requests);
  auto cost_of = [&](int64_t r) -> int64_t {
    TreeExtent e;
    if (!tree_extent(p, r, e)) return 0;
    const RequestItems q = items_of(p, e, group);
    return q.items * q.cost;
  };
  int64_t mine = 0;
  for (int64_t r = r_lo; r < r_hi; ++r) mine += cost_of(r);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) warp_sum_sh[warp] = incl;
  if (tid == 0) g.cuts[blockIdx.x].valid = 0;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const int64_t v = warp_sum_sh[w];
    if (w < warp) before += v;
    total += v;
  }
  const int64_t share = axis_share(total, gridDim.x);
  const int64_t my_lo = blockIdx.x * share, my_hi = min(my_lo + share, total);
  if (my_lo >= total) return;
  if (before <= my_lo && my_lo < before + mine) {
    int64_t r = r_lo, at = before;
    for (;; ++r) {
      const int64_t c = cost_of(r);
      if (my_lo < at + c) break;
      at += c;
    }
    start_r_sh = r;
    start_at_sh = at;
  }

  float* q_sh = sm;  // [kRowTile][kQStride]; in fp32 (hi, lo): every tile takes it
  float* k_sh = q_sh + kQParts * kRowTile * kQStride;  // [kKeyTile][kKStride]
  float* v_sh = k_sh + kKeyTile * kKStride;            // [kKeyTile][kVStride]
  float* s_sh = v_sh + kKeyTile * kVStride;  // [kRowTile][kSStride]: scores, then P
  float* corr_sh = s_sh + kRowTile * kSStride;
  // Columns behind head_dim stay 0 in every tile.
  for (int i = tid; i < kKeyTile * (kDim - dim); i += kThreads) {
    const int key = i / (kDim - dim), d = dim + i % (kDim - dim);
    k_sh[key * kKStride + d] = 0.f;
    v_sh[key * kVStride + d] = 0.f;
  }
  const T* keys = static_cast<const T*>(p.cache);
  const T* values = keys + p.num_blocks * p.block_size * p.num_kv_heads * dim;
  // MMA fragments: 16 rows from r16, keys from key16, columns from c0; fr =
  // lane / 4 and fc = lane % 4 place a lane in a fragment.
  const int r16 = 16 * (warp & 1), key16 = 16 * (warp >> 1), c0 = (warp >> 1) * 8 * NT;
  const int fr = lane >> 2, fc = lane & 3;

  __syncthreads();
  int64_t r = start_r_sh - 1, at = start_at_sh;  // request and its place on the axis
  TreeExtent e;
  RequestItems q{};
  int32_t item = 0;
#pragma unroll 1
  for (;; ++item) {
    if (item >= q.items) {  // the next request with nodes
      at += q.items * q.cost;
      if (at >= my_hi) break;
      do ++r;
      while (r < p.num_requests && !tree_extent(p, r, e));
      if (r >= p.num_requests) break;
      q = items_of(p, e, group);
      item = my_lo > at ? (int32_t)divide(my_lo - at, q.cost) : 0;
    }
    const int64_t cost0 = at + item * q.cost;
    if (cost0 >= my_hi) break;
    const int32_t j0 = (int32_t)min(max(my_lo - cost0 - kItemCost, (int64_t)0), (int64_t)q.tiles);
    const int32_t j1 = (int32_t)min(max(my_hi - cost0 - kItemCost, (int64_t)0), (int64_t)q.tiles);
    if (j0 >= j1) continue;
    __syncthreads();  // the item before is done with shared memory
    // Rows and positions fit 32 bits (a context is at most 2^30 long); 64-bit
    // divisions would cost microseconds before the first load.
    const int32_t h = item / q.row_tiles, row0 = item % q.row_tiles * kRowTile, n_rows = q.n_rows;
    const bool whole_item = j0 == 0 && j1 == q.tiles;
    const int64_t part = 2 * (int64_t)blockIdx.x + (j0 == 0 ? 1 : 0);
    if (j0 == 0 && !whole_item && tid == 0)
      g.cuts[blockIdx.x] = {e.qs, cost0, share, row0, n_rows, h, q.tiles, 1};
    const int64_t* trow = p.table + r * p.table_stride;
    const bool active = row0 + r16 < n_rows;  // this warp's MMA rows hold queries

    // Slots of tile j, by 64 threads; K or V of a tile, a warp taking every
    // eighth key, asynchronously for fp32.
    auto block_of = [&](int32_t j) -> int64_t {
      const int32_t pos = (int32_t)e.lo + j * kKeyTile + tid, lb = pos / p.block_size;
      return tid < kKeyTile && j < j1 && pos < e.hi && lb < p.table_width ? __ldg(trow + lb) : -1;
    };
    auto put_slot = [&](int32_t j, int64_t blk) {
      if (tid >= kKeyTile) return;
      const int32_t pos = (int32_t)e.lo + j * kKeyTile + tid;
      int64_t slot = -1;
      if (j < j1 && pos < e.hi) {
        if (blk >= 0 && blk < p.num_blocks)
          slot = ((blk * p.block_size + pos % p.block_size) * p.num_kv_heads + h) * dim;
        else if (p.status != nullptr)
          atomicOr(p.status, MVB_STATUS_BLOCK_OUT_OF_RANGE);
      }
      slots_sh[j & 1][tid] = slot;
    };
    auto load = [&](int32_t j, const T* from, float* to, int stride) {
      if (j < j1) {
#pragma unroll
        for (int key = warp; key < kKeyTile; key += kThreads / 32) {
          const int64_t slot = slots_sh[j & 1][key];
          if constexpr (kVec) {
#pragma unroll
            for (int c = 0; c < (kDim + 127) / 128; ++c) {
              const int d = 128 * c + 4 * lane;
              if (d >= dim) continue;
              if constexpr (kFp32)
                copy16(to + key * stride + d, from + (slot >= 0 ? slot + d : 0), slot >= 0);
              else
                *reinterpret_cast<float4*>(to + key * stride + d) =
                    slot >= 0 ? load4<T>(from + slot + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
          } else {
            for (int d = lane; d < dim; d += 32)
              to[key * stride + d] = slot >= 0 ? to_float(from[slot + d]) : 0.f;
          }
        }
      }
      copy_commit();  // a group for every call, so that the waits count alike
    };

    // The first block ids, the windows and the query rows come in together.
    const int64_t first_block = block_of(j0);
    const int32_t wrow = row0 + warp * kWarpRows;  // this warp's rows
    const int32_t lo = (int32_t)e.lo, committed = (int32_t)e.committed;
    int32_t node_of[kWarpRows], lo_row[kWarpRows];  // -1: no row
    int32_t lo_all = lo;
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i) {
      const bool ok = wrow + i < n_rows;
      node_of[i] = ok ? (wrow + i) / group : -1;
      lo_row[i] = ok ? (int32_t)min(max(e.lo, __ldg(p.qstart + e.qs + node_of[i])), e.committed) : lo;
      lo_all = max(lo_all, lo_row[i]);
    }
    float q_in[kWarpRows][NT];
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i) {
      const int32_t row = wrow + i;
      const T* src = static_cast<const T*>(p.query) + (e.qs + row / group) * p.q_st +
                     (int64_t)(h * group + row % group) * p.q_sh;
#pragma unroll
      for (int c = 0; c < NT; ++c)
        q_in[i][c] = row < n_rows && 32 * c + lane < dim ? to_float(src[32 * c + lane]) : 0.f;
    }
    put_slot(j0, first_block);
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i)
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        const int d = 32 * c + lane;
        const float x = q_in[i][c];
        const int at_q = (warp * kWarpRows + i) * kQStride + d;
        if constexpr (kFp32) {
          // (inf, x) where x has no hi + lo: its scores are not finite, and
          // the scalar loop takes x.
          uint32_t hi, lo;
          split_tf32(x, hi, lo);
          const bool odd_x = !finite(x) || !finite(__uint_as_float(hi));
          reinterpret_cast<float2*>(q_sh)[at_q] =
              make_float2(odd_x ? INFINITY : __uint_as_float(hi), odd_x ? x : __uint_as_float(lo));
        } else {
          q_sh[at_q] = x;
        }
      }
    float m[kWarpRows], l[kWarpRows], acc[NT][4];
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[c][d] = 0.f;
    __syncthreads();
    load(j0, keys, k_sh, kKStride);
    load(j0, values, v_sh, kVStride);

#pragma unroll 1
    for (int32_t j = j0; j < j1; ++j) {
      // K of the next tile comes in during this one's softmax and P.V, its V
      // during the next q.k.
      const int32_t k0 = lo + j * kKeyTile;
      const int64_t* slot_sh = slots_sh[j & 1];
      copy_wait_but_last();  // K of this tile
      __syncthreads();
      const int64_t next_block = block_of(j + 1);  // in flight during q.k

      // Scores: 16 rows x 16 keys of this warp.
      float big[4][2][4] = {}, s[2][4] = {};
      const int qa = (r16 + fr) * kQStride + fc;
      const float* kb = k_sh + (key16 + fr) * kKStride + fc;
      if (active)
#pragma unroll 4
        for (int d = 0; d < kDim; d += 8) {
          const int turn = (d >> 3) & 3;
          uint32_t ah[4], al[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at_q = qa + 8 * (i & 1) * kQStride + d + 4 * (i >> 1);
            if constexpr (kFp32) {
              const float2 x = reinterpret_cast<const float2*>(q_sh)[at_q];
              ah[i] = __float_as_uint(x.x);
              al[i] = __float_as_uint(x.y);
            } else {
              ah[i] = __float_as_uint(q_sh[at_q]);
            }
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            uint32_t bh[2], bl[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float x = kb[8 * n * kKStride + d + 4 * i];
              if constexpr (kFp32)
                split_tf32(x, bh[i], bl[i]);
              else
                bh[i] = __float_as_uint(x);
            }
            if constexpr (kFp32) {
              mma_tf32(s[n], al, bh[0], bh[1]);
              mma_tf32(s[n], ah, bl[0], bl[1]);
            }
            mma_tf32(big[turn][n], ah, bh[0], bh[1]);
          }
        }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[n][i] += (big[0][n][i] + big[1][n][i]) + (big[2][n][i] + big[3][n][i]);
      auto store_scores = [&]() {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            *reinterpret_cast<float2*>(s_sh + (r16 + fr + 8 * i) * kSStride + key16 + 8 * n + 2 * fc) =
                make_float2(s[n][2 * i], s[n][2 * i + 1]);
      };
      store_scores();
      put_slot(j + 1, next_block);
      // A score that is not finite: q or K is not (or their sum), and the
      // split product may have made NaN of an infinity.  Then plain sums.
      bool odd = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) odd |= !finite(s[i >> 2][i & 3]);
      if (__syncthreads_or(odd)) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int qr = (r16 + fr + 8 * (i >> 1)) * kQStride;
            const float* kr = k_sh + (key16 + 8 * n + 2 * fc + (i & 1)) * kKStride;
            float dot = 0.f;
#pragma unroll 1
            for (int d = 0; d < dim; ++d) {
              float x = q_sh[kQParts * (qr + d)];
              if constexpr (kFp32) {
                const float lo = q_sh[2 * (qr + d) + 1];
                x = finite(x) ? x + lo : lo;
              }
              dot = fmaf(x, kr[d], dot);
            }
            s[n][i] = dot;
          }
        store_scores();
        __syncthreads();
      }
      load(j + 1, keys, k_sh, kKStride);

      // Softmax of this warp's 4 rows, a lane at keys lane and lane + 32.
      const bool whole = k0 >= lo_all && k0 + kKeyTile <= committed &&
                         __all_sync(0xffffffffu, slot_sh[lane] >= 0 && slot_sh[lane + 32] >= 0);
      float* const rows_sh = s_sh + warp * kWarpRows * kSStride + lane;
      float y[kWarpRows][2], top[kWarpRows];
#pragma unroll
      for (int i = 0; i < kWarpRows; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) y[i][u] = rows_sh[i * kSStride + 32 * u] * g.scale_log2;
      if (!whole) {
#pragma unroll
        for (int i = 0; i < kWarpRows; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int32_t pos = k0 + 32 * u + lane, key_node = pos - committed;
            bool seen = false;
            if (node_of[i] >= 0 && slot_sh[32 * u + lane] >= 0) {
              if (key_node < 0)
                seen = pos >= lo_row[i];
              else
                seen = ((uint64_t)__ldg(p.mask + (e.qs + node_of[i]) * p.mask_words + (key_node >> 6)) >>
                        (key_node & 63)) & 1u;
            }
            if (!seen) y[i][u] = -INFINITY;
          }
      }
#pragma unroll
      for (int i = 0; i < kWarpRows; ++i) top[i] = fmaxf(y[i][0], y[i][1]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < kWarpRows; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
      for (int i = 0; i < kWarpRows; ++i) {
        const float m_new = fmaxf(m[i], top[i]), mu = m_new == -INFINITY ? 0.f : m_new;
        const float corr = exp2f(m[i] - mu);
        y[i][0] = exp2f(y[i][0] - mu);
        y[i][1] = exp2f(y[i][1] - mu);
        m[i] = m_new;
        l[i] = fmaf(l[i], corr, y[i][0] + y[i][1]);  // this lane's keys
        rows_sh[i * kSStride] = y[i][0];
        rows_sh[i * kSStride + 32] = y[i][1];
        if (lane == 0) corr_sh[warp * kWarpRows + i] = corr;
      }
      copy_wait_but_last();  // V of this tile
      __syncthreads();

      // O = O corr + P V: 16 rows x 8 NT columns of this warp.
      const float* pa = s_sh + (r16 + fr) * kSStride + fc;
      const float* vb = v_sh + fc * kVStride + c0 + fr;
      float big_t[2][NT][4] = {}, t[NT][4] = {};
      if (active)
#pragma unroll 2
        for (int k = 0; k < kKeyTile; k += 8) {
          const int turn = (k >> 3) & 1;
          const float a[4] = {pa[k], pa[8 * kSStride + k], pa[k + 4], pa[8 * kSStride + k + 4]};
          uint32_t ah[4], al[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) split_tf32(a[i], ah[i], al[i]);
#pragma unroll
          for (int c = 0; c < NT; ++c) {
            uint32_t bh[2], bl[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float x = vb[(k + 4 * i) * kVStride + 8 * c];
              if constexpr (kFp32)
                split_tf32(x, bh[i], bl[i]);
              else
                bh[i] = __float_as_uint(x);
            }
            mma_tf32(t[c], al, bh[0], bh[1]);
            if constexpr (kFp32) mma_tf32(t[c], ah, bl[0], bl[1]);
            mma_tf32(big_t[turn][c], ah, bh[0], bh[1]);
          }
        }
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[c][i] += big_t[0][c][i] + big_t[1][c][i];
      // A sum that is not finite: V holds such a value, of a key seen or not.
      bool odd_v = false;
#pragma unroll
      for (int i = 0; i < 4 * NT; ++i) odd_v |= !finite(t[i >> 2][i & 3]);
      if (__syncthreads_or(odd_v)) {
#pragma unroll
        for (int c = 0; c < NT; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* pr = s_sh + (r16 + fr + 8 * (i >> 1)) * kSStride;
            const float* vr = v_sh + c0 + 8 * c + 2 * fc + (i & 1);
            float sum = 0.f;
#pragma unroll 1
            for (int k = 0; k < kKeyTile; ++k)
              if (pr[k] != 0.f) sum = fmaf(pr[k], vr[k * kVStride], sum);  // 0: not seen
            t[c][i] = sum;
          }
        __syncthreads();
      }
      const float corr_a = corr_sh[r16 + fr], corr_b = corr_sh[r16 + fr + 8];
#pragma unroll
      for (int c = 0; c < NT; ++c) {
        acc[c][0] = fmaf(acc[c][0], corr_a, t[c][0]);
        acc[c][1] = fmaf(acc[c][1], corr_a, t[c][1]);
        acc[c][2] = fmaf(acc[c][2], corr_b, t[c][2]);
        acc[c][3] = fmaf(acc[c][3], corr_b, t[c][3]);
      }
      load(j + 1, values, v_sh, kVStride);
    }

    // Each row's (max, sum) from the warp that owns it to the warps that hold
    // its O.
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i) l[i] = warp_sum(l[i]);
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i)
      if (lane == 0) {
        s_sh[(warp * kWarpRows + i) * kSStride] = m[i];
        s_sh[(warp * kWarpRows + i) * kSStride + 1] = l[i];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int in_tile = r16 + fr + 8 * i;
      if (row0 + in_tile >= n_rows) continue;
      const int64_t row =
          (e.qs + (row0 + in_tile) / group) * p.num_q_heads + h * group + (row0 + in_tile) % group;
      const float m_row = s_sh[in_tile * kSStride], l_row = s_sh[in_tile * kSStride + 1];
      const float inv = l_row == 0.f ? 0.f : 1.f / l_row;
      if (!whole_item && c0 == 0 && fc == 0) g.part_ml[part * kRowTile + in_tile] = make_float2(m_row, l_row);
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int d = c0 + 8 * c + 2 * fc + u;
          if (d >= dim) continue;
          if (!whole_item)
            g.part_o[(part * kRowTile + in_tile) * dim + d] = acc[c][2 * i + u];
          else
            out[row * dim + d] = from_float<T>(acc[c][2 * i + u] * inv);
        }
    }
  }
}

// Joins the partials of the items that were cut, a warp per row, and writes 0
// to the rows that no request owns.  One block per SM; with as many launches as
// rows would need, and a lookup of each row's request, 5 x 48 rows x 1 tile took
// 36 us against 20.
constexpr int kJoinThreads = 1024;

template <typename T, int kLaneCols>
__global__ void __launch_bounds__(kJoinThreads, 1)
    tree_join_kernel(const TreeProblem p, const GenericParams g, int32_t ctas) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t warp0 = (int64_t)warp * gridDim.x + blockIdx.x;  // neighbours on different SMs
  const int64_t warps = (int64_t)gridDim.x * (kJoinThreads / 32);
  const int32_t dim = p.head_dim, group = p.num_q_heads / p.num_kv_heads;
  T* out = static_cast<T*>(p.out);
  // The attention before does not write these rows, and its inputs were there
  // before it began.
  for_unowned_rows(p, lane, warp0, warps, [&](int64_t t0, int64_t t1) {
    const int64_t first = t0 * p.num_q_heads * dim, last = t1 * p.num_q_heads * dim;
    for (int64_t e = first + lane; e < last; e += 32) out[e] = from_float<T>(0.f);
  });
  grid_dependency_wait();
  for (int64_t job = warp0; job < (int64_t)ctas * kRowTile; job += warps) {
    const int32_t b0 = (int32_t)(job % ctas), in_tile = (int32_t)(job / ctas);
    const CutItem c = g.cuts[b0];
    const int32_t row = c.row0 + in_tile;
    if (!c.valid || row >= c.n_rows) continue;
    // Every share from the item's first tile to its last holds some.
    const int32_t b_last = (int32_t)divide(c.cost0 + kItemCost + c.tiles - 1, c.share);
    float m = -INFINITY, l = 0.f, o[kLaneCols] = {};
#pragma unroll 2
    for (int32_t b = b0; b <= b_last; ++b) {
      const int64_t at = (2 * (int64_t)b + (b == b0 ? 1 : 0)) * kRowTile + in_tile;
      const float2 ml = __ldcg(g.part_ml + at);
      float add[kLaneCols];
#pragma unroll
      for (int k = 0; k < kLaneCols; ++k)
        add[k] = 32 * k + lane < dim ? __ldcg(g.part_o + at * dim + 32 * k + lane) : 0.f;
      const float m_new = fmaxf(m, ml.x), mu = m_new == -INFINITY ? 0.f : m_new;
      const float f0 = exp2f(m - mu), f1 = exp2f(ml.x - mu);
      m = m_new;
      l = l * f0 + ml.y * f1;
#pragma unroll
      for (int k = 0; k < kLaneCols; ++k) o[k] = o[k] * f0 + add[k] * f1;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* dst = out + ((c.qs + row / group) * p.num_q_heads + (int64_t)c.h * group + row % group) * dim;
#pragma unroll
    for (int k = 0; k < kLaneCols; ++k)
      if (32 * k + lane < dim) dst[32 * k + lane] = from_float<T>(o[k] * inv);
  }
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
struct GenericLayout {
  size_t ml, o, end;  // (the cut items come first)
};
GenericLayout generic_layout(int64_t ctas, int32_t head_dim) {
  GenericLayout w;
  w.ml = align256((size_t)ctas * sizeof(CutItem));
  w.o = align256(w.ml + (size_t)ctas * 2 * kRowTile * sizeof(float2));
  w.end = w.o + (size_t)ctas * 2 * kRowTile * head_dim * sizeof(float);
  return w;
}

template <typename T, int NT, bool kVec>
int launch(const TreeProblem& p) {
  constexpr int kDim = 32 * NT;
  constexpr int kQParts = std::is_same<T, float>::value ? 2 : 1;
  constexpr size_t kSmem = sizeof(float) * (kQParts * kRowTile * (kDim + 4) + kKeyTile * (kDim + 4) + kKeyTile * (kDim + 8) +
                                            kRowTile * (kKeyTile + 4) + kRowTile);
  static std::mutex lock;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> guard(lock);
    if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
      const cudaError_t err = cudaFuncSetAttribute(tree_attention_generic_kernel<T, NT, kVec>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
      if (err != cudaSuccess) {
        set_last_cuda_error(err);
        return MVB_ERR_CUDA;
      }
      if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
    }
  }
  // As many CTAs as the SMs hold (shared memory: two, or one of head_dim > 128).
  const int sms = num_sms() < kMaxTreeCtas ? num_sms() : kMaxTreeCtas;
  const int ctas = NT <= 4 ? 2 * sms : sms;
  const GenericLayout w = generic_layout(ctas, p.head_dim);
  if (p.workspace == nullptr || ((uintptr_t)p.workspace % 256) != 0) return MVB_ERR_INVALID_ARGUMENT;
  if (p.workspace_bytes < w.end) return MVB_ERR_WORKSPACE_TOO_SMALL;
  char* ws = static_cast<char*>(p.workspace);
  GenericParams g;
  g.scale_log2 = p.scale * 1.4426950408889634f;
  g.cuts = reinterpret_cast<CutItem*>(ws);
  g.part_ml = reinterpret_cast<float2*>(ws + w.ml);
  g.part_o = reinterpret_cast<float*>(ws + w.o);
  tree_attention_generic_kernel<T, NT, kVec><<<ctas, kThreads, kSmem, p.stream>>>(p, g);
  const int rc = check_launch();
  if (rc != MVB_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)sms);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = p.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, tree_join_kernel<T, NT>, p, g, (int32_t)ctas);
  if (err != cudaSuccess) {
    set_last_cuda_error(err);
    return MVB_ERR_CUDA;
  }
  return check_launch();
}

template <typename T>
int launch_typed(const TreeProblem& p) {
  const bool vec = p.head_dim % 4 == 0 && ((uintptr_t)p.cache % (4 * sizeof(T))) == 0;
  if (p.head_dim <= 64) return vec ? launch<T, 2, true>(p) : launch<T, 2, false>(p);
  if (p.head_dim <= 128) return vec ? launch<T, 4, true>(p) : launch<T, 4, false>(p);
  return vec ? launch<T, 8, true>(p) : launch<T, 8, false>(p);
}

}  // namespace

size_t tree_generic_workspace_bytes(int32_t head_dim) { return generic_layout(kMaxCtas, head_dim).end; }

int launch_tree_attention_generic(const TreeProblem& p) {
  if (p.head_dim > 256) return MVB_ERR_UNSUPPORTED_SHAPE;
  switch (p.dtype) {
    case MVB_DTYPE_F16:
      return launch_typed<__half>(p);
    case MVB_DTYPE_BF16:
      return launch_typed<__nv_bfloat16>(p);
    case MVB_DTYPE_F32:
      return launch_typed<float>(p);
    default:
      return MVB_ERR_UNSUPPORTED_DTYPE;
  }
}

}  // namespace mvb
