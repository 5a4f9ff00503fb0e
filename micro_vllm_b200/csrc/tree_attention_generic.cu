// Exact CUDA-core attention of draft trees over the paged cache, for every
// shape the tensor-core kernel does not take: fp32, any head_dim up to 256,
// any block size, any GQA ratio.  All arithmetic is fp32.
//
// A CTA takes 32 query rows (node, head of one GQA group) of a request and KV
// head, and walks the request's keys in tiles of 64: K and V rows come into
// shared memory once for the 32 rows, converted to fp32.  A warp owns 4 rows:
// for q.k a lane owns 2 keys (12 shared-memory wavefronts for 32 FMA
// instructions), for P.V a lane owns 4 columns per 128 (5 wavefronts for 16),
// so the bound is FMA issue and shared memory together, about half of the
// fp32 peak; the softmax statistics stay in the warp's registers.
//
// When there are fewer CTAs than the GPU holds, the key axis is cut into
// `splits` equal parts, whose (max, sum, weighted V) partials a second launch
// joins in order.  What a row does not see does not reach it: its score is
// -inf and its value is replaced by 0 (0 x NaN) in the tiles that hold keys
// not every row sees.
#include <math.h>

#include <mutex>

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
__device__ __forceinline__ float4 load4<float>(const float* at) {
  return __ldg(reinterpret_cast<const float4*>(at));
}
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

// DQ: 4-column chunks of a lane (head_dim <= 128 DQ).  kVec: cache rows are
// whole, aligned 4-element vectors.
template <typename T, int DQ, bool kVec>
__global__ void __launch_bounds__(kThreads) tree_attention_generic_kernel(const TreeProblem p,
                                                                          const GenericParams g) {
  extern __shared__ __align__(16) float sm[];
  __shared__ int64_t warp_sum_sh[kThreads / 32];
  __shared__ int64_t found_r, found_tile;
  __shared__ int64_t slot_sh[kKeyTile];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int32_t dim = p.head_dim, dim4 = (dim + 3) & ~3, group = p.num_q_heads / p.num_kv_heads;
  const int32_t h = blockIdx.y, split = blockIdx.z;
  T* out = static_cast<T*>(p.out);

  // Rows that no request owns, 32 tokens to a warp.
  if (h == 0 && split == 0) {
    for (int64_t t0 = 32 * ((int64_t)blockIdx.x * (kThreads / 32) + warp); t0 < p.num_tokens;
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
  }

  // The request and row tile of block x.
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
  if (tid == 0) found_r = -1;
  __syncthreads();
  int64_t at = incl - mine;
  for (int w = 0; w < warp; ++w) at += warp_sum_sh[w];
  if (at <= blockIdx.x && blockIdx.x < at + mine) {
    int64_t r = r_lo;
    for (;; ++r) {
      const int64_t n = row_tiles(p, r, group);
      if (blockIdx.x < at + n) break;
      at += n;
    }
    found_r = r;
    found_tile = blockIdx.x - at;
  }
  __syncthreads();
  const int64_t r = found_r;
  if (r < 0) return;
  TreeExtent e;
  tree_extent(p, r, e);
  // Rows and positions fit 32 bits (a context is at most 2^30 long); 64-bit
  // divisions would cost microseconds before the first load.
  const int32_t n_rows = (int32_t)(e.qe - e.qs) * group, row0 = (int32_t)found_tile * kRowTile;

  float* q_sh = sm;                                     // [kRowTile][dim4]
  float* k_sh = q_sh + kRowTile * dim4;                 // [kKeyTile][dim4 + 4]
  float* v_sh = k_sh + kKeyTile * (dim4 + 4);           // [kKeyTile][dim4]
  float* p_sh = v_sh + kKeyTile * dim4 + warp * kKeyTile * kWarpRows;  // this warp's [key][4 rows]
  const int32_t wrow = row0 + warp * kWarpRows;  // this warp's rows
  for (int i = 0; i < kWarpRows; ++i) {
    const int32_t row = wrow + i;
    const T* src = row < n_rows ? static_cast<const T*>(p.query) + (e.qs + row / group) * p.q_st +
                                      (int64_t)(h * group + row % group) * p.q_sh
                                : nullptr;
    for (int d = lane; d < dim4; d += 32)
      q_sh[(warp * kWarpRows + i) * dim4 + d] = src != nullptr && d < dim ? to_float(src[d]) : 0.f;
  }

  const bool active = wrow < n_rows;
  int64_t tok[kWarpRows], lo_row[kWarpRows];
  int64_t lo_all = e.lo;
#pragma unroll
  for (int i = 0; i < kWarpRows; ++i) {
    const bool ok = wrow + i < n_rows;
    tok[i] = ok ? e.qs + (wrow + i) / group : -1;
    lo_row[i] = ok ? min(max(e.lo, __ldg(p.qstart + tok[i])), e.committed) : e.lo;
    lo_all = max(lo_all, lo_row[i]);
  }
  float m[kWarpRows], l[kWarpRows], acc[DQ][kWarpRows][4];
#pragma unroll
  for (int i = 0; i < kWarpRows; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DQ; ++c)
#pragma unroll
      for (int d = 0; d < 4; ++d) acc[c][i][d] = 0.f;
  }

  const int64_t tiles = (e.hi - e.lo + kKeyTile - 1) / kKeyTile;
  const int64_t share = (tiles + g.splits - 1) / g.splits;
  const int64_t j0 = min(split * share, tiles), j1 = min(j0 + share, tiles);
  const T* cache = static_cast<const T*>(p.cache);
  const int64_t plane = p.num_blocks * p.block_size * p.num_kv_heads * dim;
  const int64_t* trow = p.table + r * p.table_stride;
  for (int64_t j = j0; j < j1; ++j) {
    const int64_t k0 = e.lo + j * kKeyTile;
    __syncthreads();  // the tile before is read
    if (tid < kKeyTile) {
      const int32_t pos = (int32_t)k0 + tid, lb = pos / p.block_size;
      int64_t slot = -1;
      if (pos < e.hi) {
        const int64_t blk = lb < p.table_width ? __ldg(trow + lb) : -1;
        if (blk >= 0 && blk < p.num_blocks)
          slot = ((blk * p.block_size + pos - lb * p.block_size) * p.num_kv_heads + h) * dim;
        else if (p.status != nullptr)
          atomicOr(p.status, MVB_STATUS_BLOCK_OUT_OF_RANGE);
      }
      slot_sh[tid] = slot;
    }
    __syncthreads();
    // A warp takes every eighth key, a lane 4 columns per 128.
    if constexpr (kVec) {
#pragma unroll 4
      for (int key = warp; key < kKeyTile; key += kThreads / 32) {
        const int64_t slot = slot_sh[key];
#pragma unroll
        for (int c = 0; c < DQ; ++c) {
          const int d = 128 * c + 4 * lane;
          if (d >= dim) continue;
          float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
          if (slot >= 0) {
            k = load4<T>(cache + slot + d);
            v = load4<T>(cache + plane + slot + d);
          }
          *reinterpret_cast<float4*>(k_sh + key * (dim4 + 4) + d) = k;
          *reinterpret_cast<float4*>(v_sh + key * dim4 + d) = v;
        }
      }
    } else {
      for (int key = warp; key < kKeyTile; key += kThreads / 32) {
        const int64_t slot = slot_sh[key];
        for (int d = lane; d < dim4; d += 32) {
          const bool ok = slot >= 0 && d < dim;
          k_sh[key * (dim4 + 4) + d] = ok ? to_float(cache[slot + d]) : 0.f;
          v_sh[key * dim4 + d] = ok ? to_float(cache[plane + slot + d]) : 0.f;
        }
      }
    }
    __syncthreads();
    if (!active) continue;

    // Scores of 4 rows x this lane's keys k0 + lane and k0 + 32 + lane.
    float s[2][kWarpRows] = {};
    const float* qr = q_sh + warp * kWarpRows * dim4;
    const float* kr = k_sh + lane * (dim4 + 4);
#pragma unroll 2
    for (int d = 0; d < dim4; d += 4) {
      const float4 ka = *reinterpret_cast<const float4*>(kr + d);
      const float4 kb = *reinterpret_cast<const float4*>(kr + 32 * (dim4 + 4) + d);
#pragma unroll
      for (int i = 0; i < kWarpRows; ++i) {
        const float4 q = *reinterpret_cast<const float4*>(qr + i * dim4 + d);
        s[0][i] = fmaf(q.w, ka.w, fmaf(q.z, ka.z, fmaf(q.y, ka.y, fmaf(q.x, ka.x, s[0][i]))));
        s[1][i] = fmaf(q.w, kb.w, fmaf(q.z, kb.z, fmaf(q.y, kb.y, fmaf(q.x, kb.x, s[1][i]))));
      }
    }
    const bool whole = k0 >= lo_all && k0 + kKeyTile <= e.committed &&
                       __all_sync(0xffffffffu, slot_sh[lane] >= 0 && slot_sh[lane + 32] >= 0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t pos = k0 + 32 * u + lane;
#pragma unroll
      for (int i = 0; i < kWarpRows; ++i) {
        bool seen = whole;
        if (!whole && tok[i] >= 0 && slot_sh[32 * u + lane] >= 0) {
          if (pos < e.committed) {
            seen = pos >= lo_row[i];
          } else {
            const int64_t node = pos - e.committed;
            seen = ((uint64_t)__ldg(p.mask + tok[i] * p.mask_words + (node >> 6)) >> (node & 63)) & 1u;
          }
        }
        s[u][i] = seen ? s[u][i] * g.scale_log2 : -INFINITY;
      }
    }
#pragma unroll
    for (int i = 0; i < kWarpRows; ++i) {
      float top = fmaxf(s[0][i], s[1][i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float m_new = fmaxf(m[i], top), mu = m_new == -INFINITY ? 0.f : m_new;
      const float corr = exp2f(m[i] - mu);
      s[0][i] = exp2f(s[0][i] - mu);
      s[1][i] = exp2f(s[1][i] - mu);
      m[i] = m_new;
      l[i] = l[i] * corr + warp_sum(s[0][i] + s[1][i]);
#pragma unroll
      for (int c = 0; c < DQ; ++c)
#pragma unroll
        for (int d = 0; d < 4; ++d) acc[c][i][d] *= corr;
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 2; ++u)
      *reinterpret_cast<float4*>(p_sh + (32 * u + lane) * kWarpRows) =
          make_float4(s[u][0], s[u][1], s[u][2], s[u][3]);
    __syncwarp();
    auto weigh = [&](bool guard) {
#pragma unroll 4
      for (int key = 0; key < kKeyTile; ++key) {
        const float4 w4 = *reinterpret_cast<const float4*>(p_sh + key * kWarpRows);
        const float w[kWarpRows] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
        for (int c = 0; c < DQ; ++c) {
          const int d0 = 128 * c + 4 * lane;
          if (d0 >= dim4) continue;
          const float4 v4 = *reinterpret_cast<const float4*>(v_sh + key * dim4 + d0);
          const float v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
          for (int i = 0; i < kWarpRows; ++i)
#pragma unroll
            for (int d = 0; d < 4; ++d) acc[c][i][d] = fmaf(w[i], guard && w[i] == 0.f ? 0.f : v[d], acc[c][i][d]);
        }
      }
    };
    if (whole)
      weigh(false);
    else
      weigh(true);
  }
  if (!active) return;

  const int64_t rows = p.num_tokens * p.num_q_heads;
#pragma unroll
  for (int i = 0; i < kWarpRows; ++i) {
    if (tok[i] < 0) continue;
    const int64_t row = tok[i] * p.num_q_heads + h * group + (wrow + i) % group;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    if (g.splits > 1 && lane == 0) g.part_ml[split * rows + row] = make_float2(m[i], l[i]);
#pragma unroll
    for (int c = 0; c < DQ; ++c)
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const int at_d = 128 * c + 4 * lane + d;
        if (at_d >= dim) continue;
        if (g.splits > 1)
          g.part_o[(split * rows + row) * dim + at_d] = acc[c][i][d];
        else
          out[row * dim + at_d] = from_float<T>(acc[c][i][d] * inv);
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

// Splits of the key axis: enough CTAs for two on each SM.
constexpr int64_t kWantCtas = 2 * 148;
int32_t splits_for(int64_t num_tokens, int64_t num_requests, int32_t num_q_heads, int32_t num_kv_heads) {
  const int64_t ctas = row_tile_bound(num_tokens, num_requests, num_q_heads / num_kv_heads) * num_kv_heads;
  if (ctas == 0) return 1;
  const int64_t want = (kWantCtas + ctas - 1) / ctas;
  return (int32_t)(want < kMaxSplits ? want : kMaxSplits);
}

template <typename T, int DQ, bool kVec>
int launch(const TreeProblem& p, const GenericParams& g, dim3 grid, size_t smem) {
  static std::mutex lock;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  {
    std::lock_guard<std::mutex> guard(lock);
    if (dev < 0 || dev >= kMaxDevices || !configured[dev]) {
      const cudaError_t err = cudaFuncSetAttribute(tree_attention_generic_kernel<T, DQ, kVec>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
      if (err != cudaSuccess) {
        set_last_cuda_error(err);
        return MVB_ERR_CUDA;
      }
      if (dev >= 0 && dev < kMaxDevices) configured[dev] = true;
    }
  }
  tree_attention_generic_kernel<T, DQ, kVec><<<grid, kThreads, smem, p.stream>>>(p, g);
  int rc = check_launch();
  if (rc != MVB_OK || g.splits == 1) return rc;
  const int64_t rows = p.num_tokens * p.num_q_heads;
  tree_join_kernel<T><<<(unsigned)((rows + 7) / 8), kThreads, 0, p.stream>>>(p, g);
  return check_launch();
}

template <typename T>
int launch_typed(const TreeProblem& p, const GenericParams& g, dim3 grid, size_t smem) {
  const bool vec = p.head_dim % 4 == 0 && ((uintptr_t)p.cache % (4 * sizeof(T))) == 0;
  if (p.head_dim <= 128)
    return vec ? launch<T, 1, true>(p, g, grid, smem) : launch<T, 1, false>(p, g, grid, smem);
  return vec ? launch<T, 2, true>(p, g, grid, smem) : launch<T, 2, false>(p, g, grid, smem);
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
  if (tiles > 0x7fffffffLL || p.num_kv_heads > 65535 ||
      (p.num_tokens * p.num_q_heads + 7) / 8 > 0x7fffffffLL)
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
  const int32_t dim4 = (p.head_dim + 3) & ~3;
  const size_t smem = sizeof(float) * ((size_t)kRowTile * dim4 + kKeyTile * (dim4 + 4) + kKeyTile * dim4 +
                                       (kThreads / 32) * kKeyTile * kWarpRows);
  const dim3 grid((unsigned)(tiles > 0 ? tiles : 1), (unsigned)p.num_kv_heads, (unsigned)g.splits);
  switch (p.dtype) {
    case MVB_DTYPE_F16:
      return launch_typed<__half>(p, g, grid, smem);
    case MVB_DTYPE_BF16:
      return launch_typed<__nv_bfloat16>(p, g, grid, smem);
    case MVB_DTYPE_F32:
      return launch_typed<float>(p, g, grid, smem);
    default:
      return MVB_ERR_UNSUPPORTED_DTYPE;
  }
}

}  // namespace mvb
