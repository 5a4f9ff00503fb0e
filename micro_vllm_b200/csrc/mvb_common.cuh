// Shared device helpers for the B200 paged-attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mvb200.h"

namespace mvb {

// Records the CUDA error of the last failed call on this host thread.
void set_last_cuda_error(cudaError_t err);

// Returns MVB_OK, or MVB_ERR_CUDA after recording the pending launch error.
int check_launch();

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Index of the request owning flattened query token `t`: the largest r in
// [0, R) with qsl[r] <= t, or -1 when t lies in no request (t >= qsl[R],
// or every request before t is empty).  Zero-length requests (qsl[r] ==
// qsl[r+1], CUDA-graph padding) are skipped because a later request with the
// same start also satisfies qsl[r] <= t.  A negative start (malformed
// metadata) also yields -1, so callers may index qstart[qsl[r]] safely.
__device__ __forceinline__ int64_t find_request(const int64_t* __restrict__ qsl, int64_t R,
                                                int64_t t) {
  int64_t lo = 0, hi = R;  // answer in [lo-1, hi-1]
  while (lo < hi) {
    int64_t mid = (lo + hi) >> 1;
    if (__ldg(qsl + mid) <= t)
      lo = mid + 1;
    else
      hi = mid;
  }
  int64_t r = lo - 1;
  if (r < 0 || t >= __ldg(qsl + r + 1) || __ldg(qsl + r) < 0) return -1;
  return r;
}

// The keys of draft-tree request r: committed positions [lo, committed), then
// drafted nodes [committed, hi).  False for a request that owns no node, or
// whose ranges or lengths do not fit together (its rows are written as 0).
struct TreeExtent {
  int64_t qs, qe, lo, committed, hi;
};
template <typename Problem>
__device__ __forceinline__ bool tree_extent(const Problem& p, int64_t r, TreeExtent& e) {
  e.qs = __ldg(p.qsl + r);
  e.qe = __ldg(p.qsl + r + 1);
  e.hi = __ldg(p.ctx_len + r);
  const int64_t n = e.qe - e.qs;
  if (n <= 0 || e.qs < 0 || e.qe > p.num_tokens || n > 64 * (int64_t)p.mask_words || e.hi < n ||
      e.hi > ((int64_t)1 << 30))
    return false;
  e.committed = e.hi - n;
  e.lo = min(max(__ldg(p.qstart + e.qs), (int64_t)0), e.committed);
  return true;
}

// a / b for a >= 0, b > 0; a 64-bit division is ~800 cycles on the way to
// the first load of a CTA.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
// Equal shares of a cost axis of `total` units for `ctas` CTAs (from 2^31
// units on the next power of two's).
__device__ __forceinline__ int64_t axis_share(int64_t total, uint32_t ctas) {
  return total < ((int64_t)1 << 31) ? (int64_t)(((uint32_t)total + ctas - 1) / ctas)
                                    : (total >> (31 - __clz((int)ctas))) + 1;
}
// Calls zero(t0, t1) by whole warps for the rows without an owner: before the
// first request, behind the last, and those of requests that do not fit.
template <typename Problem, typename Zero>
__device__ __forceinline__ void for_unowned_rows(const Problem& p, int lane, int64_t warp0, int64_t warps,
                                                 Zero zero) {
  for (int64_t r0 = 32 * warp0; r0 < p.num_requests + 2; r0 += 32 * warps) {
    const int64_t r = r0 + lane;
    int64_t z0 = 0, z1 = 0;
    if (r < p.num_requests) {
      TreeExtent e;
      if (!tree_extent(p, r, e)) z0 = e.qs, z1 = e.qe;
    } else if (r == p.num_requests) {
      z1 = p.num_requests > 0 ? __ldg(p.qsl) : p.num_tokens;
    } else if (r == p.num_requests + 1 && p.num_requests > 0) {
      z0 = __ldg(p.qsl + p.num_requests), z1 = p.num_tokens;
    }
    z0 = max(z0, (int64_t)0);
    z1 = min(z1, p.num_tokens);
    for (uint32_t todo = __ballot_sync(0xffffffffu, z0 < z1); todo != 0; todo &= todo - 1) {
      const int src = __ffs(todo) - 1;
      zero(__shfl_sync(0xffffffffu, z0, src), __shfl_sync(0xffffffffu, z1, src));
    }
  }
}

// Programmatic dependent launch (sm_90+): a kernel launched with
// programmatic stream serialization may start while the kernel before it in
// the stream still runs; grid_dependency_wait() returns once that kernel has
// completed and its writes are visible (at once for a normal launch), and
// allow_dependent_launch() lets the next such kernel start early.
__device__ __forceinline__ void grid_dependency_wait() {
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}
__device__ __forceinline__ void allow_dependent_launch() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
}

}  // namespace mvb
