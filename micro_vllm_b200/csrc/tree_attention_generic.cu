// Exact CUDA-core attention of draft trees over the paged cache, for every
// shape the tensor-core kernel does not take: fp32, any head_dim up to 256,
// any block size, any GQA ratio.
//
// One warp owns one (node, query head) row and keeps an fp32 online softmax
// over the keys its row sees, and touches no other: the committed positions
// max(ctx_start[first node], ctx_start[t]) .. C - 1, then the set bits of the
// node's ancestor mask.  A row that sees nothing is 0.
#include <math.h>

#include "mvb_common.cuh"
#include "mvb_internal.h"

namespace mvb {
namespace {

constexpr int kMaxDimPerLane = 8;  // head_dim <= 256

template <typename T>
__global__ void __launch_bounds__(128) tree_attention_generic_kernel(const TreeProblem p,
                                                                     float scale_log2) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (row >= p.num_tokens * p.num_q_heads) return;
  const int64_t t = row / p.num_q_heads;
  const int32_t hq = (int32_t)(row % p.num_q_heads);
  const int32_t h = hq / (p.num_q_heads / p.num_kv_heads);
  T* orow = static_cast<T*>(p.out) + row * p.head_dim;
  const int64_t r = find_request(p.qsl, p.num_requests, t);
  TreeExtent e;
  if (r < 0 || !tree_extent(p, r, e)) {
    for (int d = lane; d < p.head_dim; d += 32) orow[d] = from_float<T>(0.f);
    return;
  }
  float q[kMaxDimPerLane], acc[kMaxDimPerLane];
  const T* qrow = static_cast<const T*>(p.query) + t * p.q_st + (int64_t)hq * p.q_sh;
#pragma unroll
  for (int i = 0; i < kMaxDimPerLane; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < p.head_dim ? to_float(qrow[d]) : 0.f;
    acc[i] = 0.f;
  }
  const T* cache = static_cast<const T*>(p.cache);
  const int64_t plane = p.num_blocks * p.block_size * p.num_kv_heads * p.head_dim;
  const int64_t* trow = p.table + r * p.table_stride;
  float m = -INFINITY, l = 0.f;
  auto visit = [&](int64_t pos) {
    const int64_t lb = pos / p.block_size;
    const int64_t blk = lb < p.table_width ? __ldg(trow + lb) : -1;
    if (blk < 0 || blk >= p.num_blocks) {
      if (p.status != nullptr && lane == 0) atomicOr(p.status, MVB_STATUS_BLOCK_OUT_OF_RANGE);
      return;
    }
    const int64_t base = ((blk * p.block_size + pos % p.block_size) * p.num_kv_heads + h) * p.head_dim;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxDimPerLane; ++i) {
      const int d = lane + 32 * i;
      if (d < p.head_dim) dot += q[i] * to_float(cache[base + d]);
    }
    const float s = warp_sum(dot) * scale_log2;
    const float m_new = fmaxf(m, s);
    const float corr = m == m_new ? 1.f : exp2f(m - m_new);
    const float pw = s == m_new ? 1.f : exp2f(s - m_new);
    l = l * corr + pw;
#pragma unroll
    for (int i = 0; i < kMaxDimPerLane; ++i) {
      const int d = lane + 32 * i;
      const float v = d < p.head_dim ? to_float(cache[plane + base + d]) : 0.f;
      acc[i] = acc[i] * corr + pw * v;
    }
    m = m_new;
  };
  const int64_t lo = max(e.lo, __ldg(p.qstart + t));
  for (int64_t pos = lo; pos < e.committed; ++pos) visit(pos);
  const int nodes = (int)(e.hi - e.committed);
  for (int w = 0; 64 * w < nodes; ++w) {
    uint64_t bits = (uint64_t)__ldg(p.mask + t * p.mask_words + w);
    if (nodes - 64 * w < 64) bits &= (1ull << (nodes - 64 * w)) - 1;
    for (; bits != 0; bits &= bits - 1) visit(e.committed + 64 * w + __ffsll((long long)bits) - 1);
  }
  const float inv = 1.f / l;
#pragma unroll
  for (int i = 0; i < kMaxDimPerLane; ++i) {
    const int d = lane + 32 * i;
    if (d < p.head_dim) orow[d] = from_float<T>(l == 0.f ? 0.f : acc[i] * inv);
  }
}

}  // namespace

int launch_tree_attention_generic(const TreeProblem& p) {
  if (p.head_dim > 32 * kMaxDimPerLane) return MVB_ERR_UNSUPPORTED_SHAPE;
  const int64_t blocks = (p.num_tokens * p.num_q_heads + 3) / 4;
  if (blocks > 0x7fffffffLL) return MVB_ERR_UNSUPPORTED_SHAPE;
  const float scale_log2 = p.scale * 1.4426950408889634f;
  switch (p.dtype) {
    case MVB_DTYPE_F16:
      tree_attention_generic_kernel<__half><<<(unsigned)blocks, 128, 0, p.stream>>>(p, scale_log2);
      break;
    case MVB_DTYPE_BF16:
      tree_attention_generic_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, p.stream>>>(p, scale_log2);
      break;
    case MVB_DTYPE_F32:
      tree_attention_generic_kernel<float><<<(unsigned)blocks, 128, 0, p.stream>>>(p, scale_log2);
      break;
    default:
      return MVB_ERR_UNSUPPORTED_DTYPE;
  }
  return check_launch();
}

}  // namespace mvb
