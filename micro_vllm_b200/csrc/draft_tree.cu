// The integer and copy stages of a draft-tree step: tree metadata, the
// accepted path, and the move of the kept nodes' K/V rows.
//
// Request r owns rows qsl[r] .. qsl[r+1] of the flattened nodes; node i's
// parent is a node before it (or -1: a root).  Node i is written at logical
// position C_r + i of the request's pages, while its rotary position is
// C_r + depth(i): siblings share a position but not a slot.
#include "mvb_common.cuh"
#include "mvb_internal.h"

namespace mvb {
namespace {

constexpr int kTreeThreads = 128;

__device__ __forceinline__ int64_t tree_context_start(int64_t pos, int32_t kind, int64_t param) {
  if (kind == MVB_SPEC_SLIDING_WINDOW) return max(pos - param + 1, (int64_t)0);
  if (kind == MVB_SPEC_CHUNKED_LOCAL) return (pos / param) * param;
  return 0;
}

// ------------------------------------------------------------- metadata
// One CTA per request, and one more for the rows that no request owns.  The
// parents sit in shared memory; a thread owns a node and walks to its root
// twice, first counting (the depth), then setting a bit per ancestor inside
// the visible window.  The position falls by one per step of the walk, so
// the window ends it after position - start steps whatever the spec.
__global__ void __launch_bounds__(kTreeThreads) build_draft_tree_kernel(const DraftTreeArgs a) {
  __shared__ int32_t parent_sh[kMaxTreeNodes];
  const int tid = threadIdx.x;
  const int64_t T = a.num_tokens, R = a.num_requests;
  auto pad_row = [&](int64_t t) {
    a.positions[t] = 0;
    a.context_starts[t] = 0;
    a.slot_mapping[t] = -1;
    for (int w = 0; w < a.mask_words; ++w) a.ancestor_mask[t * a.mask_words + w] = 0;
  };
  if (blockIdx.x == R) {
    const int64_t lo = R > 0 ? min(max(a.qsl[0], (int64_t)0), T) : 0;
    const int64_t hi = R > 0 ? min(max(a.qsl[R], lo), T) : 0;
    for (int64_t t = tid; t < lo; t += kTreeThreads) pad_row(t);
    for (int64_t t = hi + tid; t < T; t += kTreeThreads) pad_row(t);
    return;
  }
  const int64_t r = blockIdx.x;
  const int64_t qs = a.qsl[r], qe = a.qsl[r + 1], c = a.committed[r];
  const int64_t n64 = qe - qs;
  const bool in_rows = qs >= 0 && n64 >= 0 && qe <= T;
  const bool fits = in_rows && n64 <= 64 * (int64_t)a.mask_words && c >= 0 && c + n64 <= kMaxContext;
  if (tid == 0) a.context_lengths[r] = fits ? c + n64 : 0;
  if (!fits) {
    if (tid == 0 && a.status) atomicOr(a.status, MVB_STATUS_INCONSISTENT_COUNTS);
    if (in_rows)
      for (int64_t t = qs + tid; t < qe; t += kTreeThreads) pad_row(t);
    return;
  }
  const int n = (int)n64;
  bool bad_parent = false;
  for (int i = tid; i < n; i += kTreeThreads) {
    const int64_t p = a.parents[qs + i];
    const bool ok = p >= -1 && p < i;
    bad_parent |= !ok;
    parent_sh[i] = ok ? (int32_t)p : -1;  // a parent that is no earlier node: a root
  }
  if (bad_parent && a.status) atomicOr(a.status, MVB_STATUS_BAD_PARENT);
  __syncthreads();
  for (int i = tid; i < n; i += kTreeThreads) {
    const int64_t t = qs + i;
    int depth = 0;
    for (int j = parent_sh[i]; j >= 0; j = parent_sh[j]) ++depth;
    const int64_t pos = c + depth;
    const int64_t start = tree_context_start(pos, a.spec_kind, a.spec_param);
    a.positions[t] = pos;
    a.context_starts[t] = start;
    const int64_t logical = c + i, page = logical / a.block_size;
    int64_t slot = -1;
    if (page < a.table_width) {
      const int64_t blk = a.block_table[r * a.table_stride + page];
      if (blk >= 0) slot = blk * a.block_size + logical % a.block_size;
    } else if (a.status) {
      atomicOr(a.status, MVB_STATUS_POSITION_PAST_TABLE);
    }
    a.slot_mapping[t] = slot;
    // Ancestors come in falling order, so the words are finished from the
    // last to the first.
    int64_t left = pos - start;  // steps until the window ends
    int w = a.mask_words - 1;
    uint64_t word = 0;
    int64_t* out = a.ancestor_mask + t * a.mask_words;
    for (int j = i; j >= 0 && left >= 0; j = parent_sh[j], --left) {
      for (; w > (j >> 6); --w) {
        out[w] = (int64_t)word;
        word = 0;
      }
      word |= 1ull << (j & 63);
    }
    for (; w >= 0; --w) {
      out[w] = (int64_t)word;
      word = 0;
    }
  }
}

// ------------------------------------------------------------ acceptance
// One CTA per request.  Every node i whose draft token is the target's token
// at its parent offers itself as that parent's successor (the lowest index
// wins), so the walk from node 0 is a chase through shared memory.
__global__ void __launch_bounds__(kTreeThreads) accept_draft_tree_kernel(const AcceptArgs a) {
  __shared__ int64_t target_sh[kMaxTreeNodes];
  __shared__ int32_t next_sh[kMaxTreeNodes];
  __shared__ int32_t path_sh[kMaxTreeNodes];
  __shared__ int32_t count_sh;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const int64_t qs = a.qsl[r], qe = a.qsl[r + 1];
  const int64_t n64 = qe - qs;
  const bool fits = qs >= 0 && n64 >= 0 && qe <= a.num_tokens && n64 <= kMaxTreeNodes;
  const int n = fits ? (int)n64 : 0;
  if (!fits && tid == 0 && a.status) atomicOr(a.status, MVB_STATUS_INCONSISTENT_COUNTS);
  for (int i = tid; i < n; i += kTreeThreads) {
    target_sh[i] = a.target_tokens[qs + i];
    next_sh[i] = INT32_MAX;
  }
  __syncthreads();
  bool bad_parent = false;
  for (int i = tid; i < n; i += kTreeThreads) {
    const int64_t p = a.parents[qs + i];
    if (p < -1 || p >= i) {
      bad_parent = true;
    } else if (p >= 0 && a.draft_tokens[qs + i] == target_sh[p]) {
      atomicMin(&next_sh[p], i);
    }
  }
  if (bad_parent && a.status) atomicOr(a.status, MVB_STATUS_BAD_PARENT);
  __syncthreads();
  if (tid == 0) {
    int k = 0;
    for (int p = 0; p < n && k < a.max_accepted; p = next_sh[p]) path_sh[k++] = p;
    count_sh = k;
  }
  __syncthreads();
  const int k = count_sh;
  for (int j = tid; j < a.max_accepted; j += kTreeThreads) {
    const int p = j < k ? path_sh[j] : -1;
    a.nodes[r * a.max_accepted + j] = p;
    a.tokens[r * a.max_accepted + j] = j < k ? target_sh[p] : -1;
  }
  if (tid == 0) {
    a.num_accepted[r] = k;
    a.new_lengths[r] = a.committed[r] + k;
    a.last_rows[r] = k > 0 ? qs + path_sh[k - 1] : -1;
  }
}

// -------------------------------------------------------------- KV move
// Kept node k (path[k], strictly increasing) moves from logical position
// C + path[k] to C + k in every layer and plane.  path[k] >= k, so a thread
// that owns one column of the row and goes through k in order reads every
// source before a store reaches it: no barrier between reads and writes.
template <typename Vec>
__global__ void __launch_bounds__(256) compact_draft_kv_kernel(const CompactArgs a) {
  extern __shared__ int64_t slot_sh[];  // [max_accepted] sources, then targets
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x;
  const int64_t kept = a.num_accepted[r], c = a.committed[r];
  int64_t* src = slot_sh;
  int64_t* dst = slot_sh + a.max_accepted;
  int bits = 0;
  if (kept < 0 || kept > a.max_accepted || c < 0 || c > kMaxContext) bits = MVB_STATUS_INCONSISTENT_COUNTS;
  const int k_all = bits ? 0 : (int)kept;
  for (int k = tid; k < k_all; k += blockDim.x) {
    const int64_t node = a.nodes[r * a.max_accepted + k];
    const int64_t before = k > 0 ? a.nodes[r * a.max_accepted + k - 1] : -1;
    if (node <= before || node >= kMaxTreeNodes) {
      bits |= MVB_STATUS_INCONSISTENT_COUNTS;
      continue;
    }
    auto slot_of = [&](int64_t logical) -> int64_t {
      const int64_t page = logical / a.block_size;
      if (page >= a.table_width) {
        bits |= MVB_STATUS_POSITION_PAST_TABLE;
        return -1;
      }
      const int64_t blk = a.block_table[r * a.table_stride + page];
      if (blk < 0 || blk >= a.num_blocks) {
        bits |= MVB_STATUS_BLOCK_OUT_OF_RANGE;
        return -1;
      }
      return blk * a.block_size + logical % a.block_size;
    };
    src[k] = node == k ? -1 : slot_of(c + node);
    dst[k] = node == k ? -1 : slot_of(c + k);
  }
  if (bits && a.status) atomicOr(a.status, bits);
  // A request with a bad entry is left as it was, in every layer.
  if (__syncthreads_or(bits)) return;
  const int64_t row_vecs = a.row_vecs;
  const int64_t plane = a.num_blocks * a.block_size * row_vecs;
  const int64_t columns = 2 * row_vecs;
  for (int layer = blockIdx.y; layer < a.num_layers; layer += gridDim.y) {
    Vec* cache = static_cast<Vec*>(a.layers[layer]);
    for (int64_t col = tid; col < columns; col += blockDim.x) {
      Vec* base = cache + (col >= row_vecs ? plane + (col - row_vecs) : col);
      for (int k = 0; k < k_all; ++k)
        if (src[k] >= 0) base[dst[k] * row_vecs] = base[src[k] * row_vecs];
    }
  }
}

}  // namespace

int launch_build_draft_tree(const DraftTreeArgs& a) {
  build_draft_tree_kernel<<<(unsigned)(a.num_requests + 1), kTreeThreads, 0, a.stream>>>(a);
  return check_launch();
}

int launch_accept_draft_tree(const AcceptArgs& a) {
  accept_draft_tree_kernel<<<(unsigned)a.num_requests, kTreeThreads, 0, a.stream>>>(a);
  return check_launch();
}

int launch_compact_draft_kv(CompactArgs a, int64_t row_bytes, bool aligned16) {
  const size_t smem = (size_t)2 * a.max_accepted * sizeof(int64_t);
  const dim3 grid((unsigned)a.num_requests, (unsigned)a.num_layers);
  if (aligned16 && row_bytes % 16 == 0) {
    a.row_vecs = row_bytes / 16;
    compact_draft_kv_kernel<uint4><<<grid, 256, smem, a.stream>>>(a);
  } else {
    a.row_vecs = row_bytes / 2;
    compact_draft_kv_kernel<uint16_t><<<grid, 256, smem, a.stream>>>(a);
  }
  return check_launch();
}

}  // namespace mvb
