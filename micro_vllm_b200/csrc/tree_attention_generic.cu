// Attention of draft trees over the paged cache for every shape that the
// tcgen05 kernel does not take: fp32, any head_dim up to 256, any block size,
// any GQA ratio.
//
// A CTA takes 32 query rows (node, head of one GQA group) of a request and KV
// head, and walks the request's keys in tiles of 64: K and V rows come into
// shared memory once for the 32 rows, as fp32.  q.k and P.V run on the tensor
// cores (mma.sync, TF32 operands, fp32 sums) with fp32 accuracy: a value is
// hi + lo, both TF32 (22 bits), and a product hi hi + hi lo + lo hi.  fp16 and
// bf16 values have no lo.  The tensor cores cut off what a sum cannot hold, half
// a last bit each time on average, so the hi products go round several sums (4
// for q.k, 2 for P.V) and the small ones have their own: one sum for all was
// 1.4e-6 off at 24 x 1.5K keys, against 5e-7 of a plain fp32 product.  On the CUDA cores the same tiles are bound by
// shared memory (12-18 TFLOP/s; two operand loads for 32 FMA instructions).
// The softmax is fp32, a warp owning 4 rows, their statistics in registers.
// Tiles that hold infinities or NaN go through scalar loops: hi and lo of an
// infinity are no sum, and what a row does not see must not reach it as 0 x NaN.
//
// When there are fewer CTAs than the GPU holds, the key axis is cut into
// `splits` equal parts, whose (max, sum, weighted V) partials a second launch
// joins in order.
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
constexpr int kMaxSplits = 32;

struct GenericParams {
  int32_t splits;
  float scale_log2;
  float* part_o;    // [splits][row][head_dim]
  float2* part_ml;  // [splits][row] (max, sum)
};

// Row tiles of request r (0 when it owns no node).
__device__ __forceinline__ int64_t row_tiles(const TreeProblem& p, int64_t r, int32_t group) {
  TreeExtent e;
  if (!tree_extent(p, r, e)) return 0;
  return ((int32_t)(e.qe - e.qs) * group + kRowTile - 1) / kRowTile;
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

// x = hi + lo, each rounded to TF32 (10 mantissa bits): 22 bits of x.  Integer
// rounding, since conversions run at a quarter of the rate.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
  lo = (__float_as_uint(x - __uint_as_float(hi)) + 0x1000u) & 0xffffe000u;
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
  constexpr int kSStride = kKeyTile + 4;
  constexpr bool kFp32 = std::is_same<T, float>::value;    // q, k and v have a lo
  extern __shared__ __align__(16) float sm[];
  __shared__ int64_t warp_sum_sh[kThreads / 32];
  __shared__ int64_t found_r, found_tile;
  __shared__ int64_t slots_sh[2][kKeyTile];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t dim = p.head_dim, group = p.num_q_heads / p.num_kv_heads;
  T* out = static_cast<T*>(p.out);

  // Rows that no request owns, 32 tokens to a warp.
  for (int64_t t0 = 32 * ((int64_t)warp * gridDim.x + blockIdx.x); t0 < p.num_tokens;
       t0 += 32 * (int64_t)gridDim.x * (kThreads / 32)) {
    const int64_t t = t0 + lane;
    bool zero = false;
    if (t < p.num_tokens) {
      const int64_t r = find_request(p.qsl, p.num_requests, t);
      TreeExtent e;
      zero = r < 0 || !tree_extent(p, r, e);
    }
    for (uint32_t todo = __ballot_sync(0xffffffffu, zero); todo != 0; todo &= todo - 1)
      for (int64_t d = lane; d < (int64_t)p.num_q_heads * dim; d += 32)
        out[(t0 + __ffs(todo) - 1) * p.num_q_heads * dim + d] = from_float<T>(0.f);
  }

  // Row tiles of all requests, counted once; an item is (row tile, KV head,
  // split), and a CTA takes every gridDim.x-th.
  const int64_t per = (p.num_requests + kThreads - 1) / kThreads;
  const int64_t r_lo = min(tid * per, p.num_requests), r_hi = min(r_lo + per, p.num_requests);
  int64_t mine = 0;
  for (int64_t r = r_lo; r < r_hi; ++r) mine += row_tiles(p, r, group);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += u;
  }
  if (lane == 31) warp_sum_sh[warp] = incl;
  __syncthreads();
  int64_t first = incl - mine, all = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) first += warp_sum_sh[w];
    all += warp_sum_sh[w];
  }

  float* q_sh = sm;                          // [kRowTile][kQStride]
  float* k_sh = q_sh + kRowTile * kQStride;  // [kKeyTile][kQStride]
  float* v_sh = k_sh + kKeyTile * kQStride;  // [kKeyTile][kVStride]
  float* s_sh = v_sh + kKeyTile * kVStride;  // [kRowTile][kSStride]: scores, then P
  float* corr_sh = s_sh + kRowTile * kSStride;
  // Columns behind head_dim stay 0 in every tile.
  for (int i = tid; i < kKeyTile * (kDim - dim); i += kThreads) {
    const int key = i / (kDim - dim), d = dim + i % (kDim - dim);
    k_sh[key * kQStride + d] = 0.f;
    v_sh[key * kVStride + d] = 0.f;
  }
  const T* keys = static_cast<const T*>(p.cache);
  const T* values = keys + p.num_blocks * p.block_size * p.num_kv_heads * dim;
  const int64_t rows = p.num_tokens * p.num_q_heads;
  // MMA fragments: 16 rows from r16, keys from key16, columns from c0; fr =
  // lane / 4 and fc = lane % 4 place a lane in a fragment.
  const int r16 = 16 * (warp & 1), key16 = 16 * (warp >> 1), c0 = (warp >> 1) * 8 * NT;
  const int fr = lane >> 2, fc = lane & 3;

  const uint32_t items = (uint32_t)all * (uint32_t)(p.num_kv_heads * g.splits);
#pragma unroll 1
  for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int32_t split = item % (uint32_t)g.splits;
    const int32_t h = item / (uint32_t)g.splits % (uint32_t)p.num_kv_heads;
    const int64_t x = item / (uint32_t)(g.splits * p.num_kv_heads);
    __syncthreads();  // the item before is done with shared memory
    if (first <= x && x < first + mine) {
      int64_t r = r_lo, at = first;
      for (;; ++r) {
        const int64_t n = row_tiles(p, r, group);
        if (x < at + n) break;
        at += n;
      }
      found_r = r;
      found_tile = x - at;
    }
    __syncthreads();
    const int64_t r = found_r;
    TreeExtent e;
    tree_extent(p, r, e);
    // Rows and positions fit 32 bits (a context is at most 2^30 long); 64-bit
    // divisions would cost microseconds before the first load.
    const int32_t n_rows = (int32_t)(e.qe - e.qs) * group, row0 = (int32_t)found_tile * kRowTile;
    const int32_t tiles = ((int32_t)(e.hi - e.lo) + kKeyTile - 1) / kKeyTile;
    const int32_t share = (tiles + g.splits - 1) / g.splits;
    const int32_t j0 = min(split * share, tiles), j1 = min(j0 + share, tiles);
    const int64_t* trow = p.table + r * p.table_stride;

    // Slots of tile j, by 64 threads; K or V of a tile, a warp taking every
    // eighth key, asynchronously for fp32.
    auto look_up = [&](int32_t j) {
      const int32_t pos = (int32_t)e.lo + j * kKeyTile + tid, lb = pos / p.block_size;
      int64_t slot = -1;
      if (j < j1 && pos < e.hi) {
        const int64_t blk = lb < p.table_width ? __ldg(trow + lb) : -1;
        if (blk >= 0 && blk < p.num_blocks)
          slot = ((blk * p.block_size + pos - lb * p.block_size) * p.num_kv_heads + h) * dim;
        else if (p.status != nullptr)
          atomicOr(p.status, MVB_STATUS_BLOCK_OUT_OF_RANGE);
      }
      slots_sh[j & 1][tid] = slot;
    };
    auto load = [&](int32_t j, const T* from, float* to, int stride) {
      if (j < j1) {
#pragma unroll 4
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

    if (tid < kKeyTile) look_up(j0);
    const int32_t wrow = row0 + warp * kWarpRows;  // this warp's rows
    for (int i = 0; i < kWarpRows; ++i) {
      const int32_t row = wrow + i;
      const T* src = row < n_rows ? static_cast<const T*>(p.query) + (e.qs + row / group) * p.q_st +
                                        (int64_t)(h * group + row % group) * p.q_sh
                                  : nullptr;
      for (int d = lane; d < kDim; d += 32)
        q_sh[(warp * kWarpRows + i) * kQStride + d] = src != nullptr && d < dim ? to_float(src[d]) : 0.f;
    }
    int64_t tok[kWarpRows], lo_row[kWarpRows];
    int64_t lo_all = e.lo;
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i) {
      const bool ok = wrow + i < n_rows;
      tok[i] = ok ? e.qs + (wrow + i) / group : -1;
      lo_row[i] = ok ? min(max(e.lo, __ldg(p.qstart + tok[i])), e.committed) : e.lo;
      lo_all = max(lo_all, lo_row[i]);
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
    load(j0, keys, k_sh, kQStride);
    load(j0, values, v_sh, kVStride);

#pragma unroll 1
    for (int32_t j = j0; j < j1; ++j) {
      // K of the next tile comes in during this one's softmax and P.V, its V
      // during the next q.k.
      const int64_t k0 = e.lo + (int64_t)j * kKeyTile;
      const int64_t* slot_sh = slots_sh[j & 1];
      copy_wait_but_last();  // K of this tile
      __syncthreads();
      if (tid < kKeyTile) look_up(j + 1);

      // Scores: 16 rows x 16 keys of this warp.
      float big[4][2][4] = {}, s[2][4] = {};
      const float* qa = q_sh + (r16 + fr) * kQStride + fc;
      const float* kb = k_sh + (key16 + fr) * kQStride + fc;
#pragma unroll 4
      for (int d = 0; d < kDim; d += 8) {
        const int turn = (d >> 3) & 3;
        const float a[4] = {qa[d], qa[8 * kQStride + d], qa[d + 4], qa[8 * kQStride + d + 4]};
        uint32_t ah[4], al[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) split_tf32(a[i], ah[i], al[i]);
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          uint32_t bh[2], bl[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) split_tf32(kb[8 * n * kQStride + d + 4 * i], bh[i], bl[i]);
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
            const float* qr = q_sh + (r16 + fr + 8 * (i >> 1)) * kQStride;
            const float* kr = k_sh + (key16 + 8 * n + 2 * fc + (i & 1)) * kQStride;
            float dot = 0.f;
#pragma unroll 1
            for (int d = 0; d < dim; ++d) dot = fmaf(qr[d], kr[d], dot);
            s[n][i] = dot;
          }
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float2*>(s_sh + (r16 + fr + 8 * i) * kSStride + key16 + 8 * n + 2 * fc) =
              make_float2(s[n][2 * i], s[n][2 * i + 1]);
      __syncthreads();
      load(j + 1, keys, k_sh, kQStride);

      // Softmax of this warp's 4 rows, a lane at keys lane and lane + 32.
      const bool whole = k0 >= lo_all && k0 + kKeyTile <= e.committed &&
                         __all_sync(0xffffffffu, slot_sh[lane] >= 0 && slot_sh[lane + 32] >= 0);
#pragma unroll
      for (int i = 0; i < kWarpRows; ++i) {
        float* row = s_sh + (warp * kWarpRows + i) * kSStride;
        float y[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int64_t pos = k0 + 32 * u + lane;
          bool seen = whole;
          if (!whole && tok[i] >= 0 && slot_sh[32 * u + lane] >= 0) {
            if (pos < e.committed) {
              seen = pos >= lo_row[i];
            } else {
              const int64_t node = pos - e.committed;
              seen = ((uint64_t)__ldg(p.mask + tok[i] * p.mask_words + (node >> 6)) >> (node & 63)) & 1u;
            }
          }
          y[u] = seen ? row[32 * u + lane] * g.scale_log2 : -INFINITY;
        }
        float top = fmaxf(y[0], y[1]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m[i], top), mu = m_new == -INFINITY ? 0.f : m_new;
        const float corr = exp2f(m[i] - mu);
        y[0] = exp2f(y[0] - mu);
        y[1] = exp2f(y[1] - mu);
        m[i] = m_new;
        l[i] = l[i] * corr + warp_sum(y[0] + y[1]);
        row[lane] = y[0];
        row[32 + lane] = y[1];
        if (lane == 0) corr_sh[warp * kWarpRows + i] = corr;
      }
      copy_wait_but_last();  // V of this tile
      __syncthreads();

      // O = O corr + P V: 16 rows x 8 NT columns of this warp.
      const float* pa = s_sh + (r16 + fr) * kSStride + fc;
      const float* vb = v_sh + fc * kVStride + c0 + fr;
      float big_t[2][NT][4] = {}, t[NT][4] = {};
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
          for (int i = 0; i < 2; ++i) split_tf32(vb[(k + 4 * i) * kVStride + 8 * c], bh[i], bl[i]);
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
      if (g.splits > 1 && c0 == 0 && fc == 0) g.part_ml[split * rows + row] = make_float2(m_row, l_row);
#pragma unroll
      for (int c = 0; c < NT; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int d = c0 + 8 * c + 2 * fc + u;
          if (d >= dim) continue;
          if (g.splits > 1)
            g.part_o[(split * rows + row) * dim + d] = acc[c][2 * i + u];
          else
            out[row * dim + d] = from_float<T>(acc[c][2 * i + u] * inv);
        }
    }
  }
}

// One warp per owned row: joins the row's splits in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) tree_join_kernel(const TreeProblem p, const GenericParams g) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = p.num_tokens * p.num_q_heads;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int64_t r = find_request(p.qsl, p.num_requests, row / p.num_q_heads);
  TreeExtent e;
  if (r < 0 || !tree_extent(p, r, e)) return;  // written as 0 before
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < g.splits) ml = __ldcg(g.part_ml + lane * rows + row);
  float top = ml.x;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float f = exp2f(ml.x - (top == -INFINITY ? 0.f : top));
  const float l = warp_sum(ml.y * f);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  for (int d0 = 0; d0 < p.head_dim; d0 += 32) {
    const int d = d0 + lane;
    float acc = 0.f;
#pragma unroll 4
    for (int s = 0; s < g.splits; ++s) {
      const float fs = __shfl_sync(0xffffffffu, f, s), ls = __shfl_sync(0xffffffffu, ml.y, s);
      if (d < p.head_dim && ls != 0.f) acc = fmaf(__ldcg(g.part_o + (s * rows + row) * p.head_dim + d), fs, acc);
    }
    if (d < p.head_dim) static_cast<T*>(p.out)[row * p.head_dim + d] = from_float<T>(acc * inv);
  }
}

// Row tiles of a batch: at most T G / 32 and one more for each request with
// a node.
int64_t row_tile_bound(int64_t num_tokens, int64_t num_requests, int32_t group) {
  const int64_t requests = num_requests < num_tokens ? num_requests : num_tokens;
  return num_tokens * group / kRowTile + requests;
}

// Splits of the key axis: enough CTAs for two on each SM.  Measured in fp32: 2,
// 4 and 8 CTAs an SM give 158, 192 and 187 us at 1 x 64 nodes x 8K keys and 46,
// 50 and 60 us at 5 x 12 nodes x 1.5K keys.
constexpr int64_t kWantCtas = 2 * 148;
int32_t splits_for(int64_t num_tokens, int64_t num_requests, int32_t num_q_heads, int32_t num_kv_heads) {
  const int64_t ctas = row_tile_bound(num_tokens, num_requests, num_q_heads / num_kv_heads) * num_kv_heads;
  if (ctas == 0) return 1;
  const int64_t want = (kWantCtas + ctas - 1) / ctas;
  return (int32_t)(want < kMaxSplits ? want : kMaxSplits);
}

template <typename T, int NT, bool kVec>
int launch(const TreeProblem& p, const GenericParams& g, dim3 grid) {
  constexpr int kDim = 32 * NT;
  constexpr size_t kSmem = sizeof(float) * (kRowTile * (kDim + 4) + kKeyTile * (kDim + 4) + kKeyTile * (kDim + 8) +
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
  tree_attention_generic_kernel<T, NT, kVec><<<grid, kThreads, kSmem, p.stream>>>(p, g);
  int rc = check_launch();
  if (rc != MVB_OK || g.splits == 1) return rc;
  const int64_t rows = p.num_tokens * p.num_q_heads;
  tree_join_kernel<T><<<(unsigned)((rows + 7) / 8), kThreads, 0, p.stream>>>(p, g);
  return check_launch();
}

template <typename T>
int launch_typed(const TreeProblem& p, const GenericParams& g, dim3 grid) {
  const bool vec = p.head_dim % 4 == 0 && ((uintptr_t)p.cache % (4 * sizeof(T))) == 0;
  if (p.head_dim <= 64) return vec ? launch<T, 2, true>(p, g, grid) : launch<T, 2, false>(p, g, grid);
  if (p.head_dim <= 128) return vec ? launch<T, 4, true>(p, g, grid) : launch<T, 4, false>(p, g, grid);
  return vec ? launch<T, 8, true>(p, g, grid) : launch<T, 8, false>(p, g, grid);
}

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

}  // namespace

// splits x rows is largest for a batch that is split: rows <= 32 x CTAs (a
// row tile holds 32 of them), so splits x rows <= (kWantCtas / CTAs + 1) rows
// <= 32 kWantCtas + rows, with CTAs < kWantCtas.
size_t tree_generic_workspace_bytes(int64_t num_tokens, int32_t num_q_heads, int32_t head_dim) {
  const int64_t rows = num_tokens * num_q_heads, most = kRowTile * kWantCtas;
  const size_t n = (size_t)(most + (rows < most ? rows : most));
  return align256(n * sizeof(float2)) + n * head_dim * sizeof(float) + 256;
}

int launch_tree_attention_generic(const TreeProblem& p) {
  if (p.head_dim > 256) return MVB_ERR_UNSUPPORTED_SHAPE;
  const int32_t group = p.num_q_heads / p.num_kv_heads;
  const int64_t tiles = row_tile_bound(p.num_tokens, p.num_requests, group);
  if (tiles > 0x7fffffffLL || (p.num_tokens * p.num_q_heads + 7) / 8 > 0x7fffffffLL)
    return MVB_ERR_UNSUPPORTED_SHAPE;
  GenericParams g;
  g.splits = splits_for(p.num_tokens, p.num_requests, p.num_q_heads, p.num_kv_heads);
  g.scale_log2 = p.scale * 1.4426950408889634f;
  const int64_t rows = p.num_tokens * p.num_q_heads;
  const size_t ml = align256((size_t)g.splits * rows * sizeof(float2));
  const size_t need = ml + (size_t)g.splits * rows * p.head_dim * sizeof(float);
  if (g.splits > 1) {
    if (p.workspace == nullptr || ((uintptr_t)p.workspace % 256) != 0) return MVB_ERR_INVALID_ARGUMENT;
    if (p.workspace_bytes < need) return MVB_ERR_WORKSPACE_TOO_SMALL;
  }
  g.part_ml = static_cast<float2*>(p.workspace);
  g.part_o = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + ml);
  const int64_t items = tiles * p.num_kv_heads * g.splits, most = 2 * (int64_t)num_sms();
  if (items > 0x7fffffffLL) return MVB_ERR_UNSUPPORTED_SHAPE;
  const dim3 grid((unsigned)(items < 1 ? 1 : items < most ? items : most));
  switch (p.dtype) {
    case MVB_DTYPE_F16:
      return launch_typed<__half>(p, g, grid);
    case MVB_DTYPE_BF16:
      return launch_typed<__nv_bfloat16>(p, g, grid);
    case MVB_DTYPE_F32:
      return launch_typed<float>(p, g, grid);
    default:
      return MVB_ERR_UNSUPPORTED_DTYPE;
  }
}

}  // namespace mvb
