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
// Block ids from here on are no pages (their slots could wrap to a real one).
constexpr int64_t kMaxBlockId = (int64_t)1 << 32;

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
// A request that does not fit pads what it claims of the rows.  Bound by
// latency: 3.2 us captured at 1 x 8 nodes, 3.9 at 256 x 64 with a window.
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
  const bool fits = qs >= 0 && n64 >= 0 && qe <= T && n64 <= 64 * (int64_t)a.mask_words && c >= 0 &&
                    c <= kMaxContext - n64;
  if (tid == 0) a.context_lengths[r] = fits ? c + n64 : 0;
  if (!fits) {
    if (tid == 0 && a.status) atomicOr(a.status, MVB_STATUS_INCONSISTENT_COUNTS);
    const int64_t end = min(qe, T);
    for (int64_t t = max(qs, (int64_t)0) + tid; t < end; t += kTreeThreads) pad_row(t);
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
      if (blk >= 0 && blk < kMaxBlockId) slot = blk * a.block_size + logical % a.block_size;
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
// wins), so the walk from node 0 is a chase through shared memory.  Bound by
// latency: 3.4 us captured at 4 x 16 and at 512 x 64 nodes.
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
// source before a store reaches it: no barrier between reads and writes, and
// kMoveBatch rows are loaded before the first of them is stored.  The bound is
// HBM (a row is read once and written once); a block takes a few layers so
// that the slot lookups (three dependent loads) are paid once for them.
// Measured at 1149 rows of 2 KB in 28 layers (264 MB): 46.9 us = 5650 GB/s;
// rows x layers of 4 x 4, 8 x 4, 4 x 2 and 4 x 7 give 46.7, 46.2, 45.5 and 48.5.
constexpr int kMoveBatch = 4, kMoveLayers = 4;

template <typename Vec>
__global__ void __launch_bounds__(256) compact_draft_kv_kernel(const CompactArgs a) {
  extern __shared__ int64_t slot_sh[];  // [max_accepted] sources, then targets
  __shared__ int32_t moves_sh;
  const int64_t r = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  int64_t* src = slot_sh;
  int64_t* dst = slot_sh + a.max_accepted;
  // One warp lists the rows that move, in order; -1 rows for a request with a
  // bad entry, which is left as it was in every layer.
  if (tid < 32) {
    const int64_t kept = a.num_accepted[r], c = a.committed[r];
    int bits = 0;
    if (kept < 0 || kept > a.max_accepted || c < 0 || c > kMaxContext) bits = MVB_STATUS_INCONSISTENT_COUNTS;
    const int k_all = bits ? 0 : (int)kept;
    auto slot_of = [&](int32_t logical) -> int64_t {
      const int32_t page = logical / (int32_t)a.block_size;
      if (page >= a.table_width) {
        bits |= MVB_STATUS_POSITION_PAST_TABLE;
        return -1;
      }
      const int64_t blk = a.block_table[r * a.table_stride + page];
      if (blk < 0 || blk >= a.num_blocks) {
        bits |= MVB_STATUS_BLOCK_OUT_OF_RANGE;
        return -1;
      }
      return blk * a.block_size + (logical - page * (int32_t)a.block_size);
    };
    int moves = 0;
    int64_t last = -1;  // node of the 32 before
    for (int k0 = 0; k0 < k_all; k0 += 32) {
      const int k = k0 + lane;
      const int64_t node = k < k_all ? a.nodes[r * a.max_accepted + k] : 0;
      int64_t before = __shfl_up_sync(0xffffffffu, node, 1);
      if (lane == 0) before = last;
      last = __shfl_sync(0xffffffffu, node, 31);
      bool move = false;
      int64_t from = -1, to = -1;
      if (k < k_all) {
        if (node <= before || node >= kMaxTreeNodes) {
          bits |= MVB_STATUS_INCONSISTENT_COUNTS;
        } else if (node != k) {
          move = true;
          from = slot_of((int32_t)(c + node));
          to = slot_of((int32_t)c + k);
        }
      }
      const uint32_t m = __ballot_sync(0xffffffffu, move);
      if (move) {
        const int at = moves + __popc(m & ((1u << lane) - 1u));
        src[at] = from * a.row_vecs;
        dst[at] = to * a.row_vecs;
      }
      moves += __popc(m);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) bits |= __shfl_xor_sync(0xffffffffu, bits, o);
    if (lane == 0) {
      if (bits && a.status) atomicOr(a.status, bits);
      moves_sh = bits ? 0 : moves;
    }
  }
  __syncthreads();
  const int moves = moves_sh;
  const int64_t row_vecs = a.row_vecs;
  const int64_t plane = a.num_blocks * a.block_size * row_vecs;
  const int layer0 = blockIdx.y * a.layers_per_block;
  const int layer1 = min(layer0 + a.layers_per_block, a.num_layers);
  for (int64_t col = tid; col < 2 * row_vecs; col += blockDim.x) {
    const int64_t at = col >= row_vecs ? plane + (col - row_vecs) : col;
    for (int k0 = 0; k0 < moves; k0 += kMoveBatch) {
#pragma unroll 2
      for (int layer = layer0; layer < layer1; ++layer) {
        Vec* base = static_cast<Vec*>(a.layers[layer]) + at;
        Vec v[kMoveBatch];
#pragma unroll
        for (int u = 0; u < kMoveBatch; ++u)
          if (k0 + u < moves) v[u] = base[src[k0 + u]];
#pragma unroll
        for (int u = 0; u < kMoveBatch; ++u)
          if (k0 + u < moves) base[dst[k0 + u]] = v[u];
      }
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
  // One layer to a block while that leaves SMs idle.
  const int64_t blocks = a.num_requests * a.num_layers / (4 * (int64_t)num_sms());
  a.layers_per_block = blocks < 1 ? 1 : blocks > kMoveLayers ? kMoveLayers : (int32_t)blocks;
  const dim3 grid((unsigned)a.num_requests,
                  (unsigned)((a.num_layers + a.layers_per_block - 1) / a.layers_per_block));
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
