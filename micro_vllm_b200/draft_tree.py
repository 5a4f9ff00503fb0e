"""Draft trees: one speculative-decoding step over the paged cache.

A step verifies a tree of drafted tokens per request instead of taking one
token.  The reference has no such step (its decode takes one token per
request, src/micro_vllm/worker/model_runner.py:724-900); these stages stand
beside the ones it has and keep everything on the device, so steps follow
each other without a host round trip:

    tree = build_draft_tree(parents, starts, committed, block_table, block_size, max_nodes=64)
    # per layer: prologue (or write_kv_cache) with tree.attention, then
    out = operator.attend_tree(query, layer_kv_cache, tree)
    # the target's token at every node: sample_tokens(logits of every node, ...)
    kept = accept_draft_tree(draft_tokens, target_tokens, parents, starts, committed, max_accepted=8)
    compactor(block_table, committed, kept.nodes, kept.num_accepted)   # DraftKVCompactor(layer caches)
    committed = kept.committed_lengths

Node 0 of a request is its pending token: the one sampled last, whose K/V is
not in the cache yet.  Node i is cached at logical position committed + i and
rotated at committed + depth(i).
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from micro_vllm_b200 import _lib
from micro_vllm_b200.attention import AttentionMetadata, FullAttentionSpec
from micro_vllm_b200.metadata import spec_code

MAX_TREE_NODES = _lib.MVB_MAX_TREE_NODES
_FULL = FullAttentionSpec()
_CACHE_DTYPES = {
    torch.float16: _lib.MVB_DTYPE_F16,
    torch.bfloat16: _lib.MVB_DTYPE_BF16,
    torch.float32: _lib.MVB_DTYPE_F32,
}


@dataclass(frozen=True, slots=True, eq=False)
class DraftTree:
    """One step's draft trees as the attention reads them: ``attention`` with
    a row per drafted node (``context_lengths`` counts the nodes too), and
    ``ancestor_mask`` int64 [rows, words]: bit j % 64 of word j / 64 says that
    the row's node sees node j of its request."""

    attention: AttentionMetadata
    ancestor_mask: torch.Tensor


@dataclass(frozen=True, slots=True, eq=False)
class AcceptedDraft:
    """What the target model keeps of each request's tree (int64, on the
    device): ``nodes`` [requests, max_accepted] and ``tokens`` (-1 behind the
    kept ones), ``num_accepted``, the new ``committed_lengths`` and
    ``last_rows``, the row of the last kept node (-1 without nodes)."""

    nodes: torch.Tensor
    num_accepted: torch.Tensor
    tokens: torch.Tensor
    committed_lengths: torch.Tensor
    last_rows: torch.Tensor


def launch(entry, device: torch.device, what: str, *args) -> None:
    """Calls a C entry whose last argument is the stream, with ``device``
    current and on its current stream, and raises for its status."""

    if torch._C._cuda_getDevice() == device.index:
        rc = entry(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            rc = entry(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if rc != _lib.MVB_OK:
        _lib.check(rc, what)


def _vector(name: str, t: torch.Tensor, device: torch.device, size: int | None = None) -> torch.Tensor:
    if t.dtype is not torch.int64 or t.dim() != 1 or t.get_device() != device.index \
            or (size is not None and t.shape[0] != size):
        raise ValueError(f"{name} must be torch.int64 [{'rows' if size is None else size}] on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _table(table: torch.Tensor, device: torch.device, requests: int) -> torch.Tensor:
    if table.dtype is not torch.int64 or table.dim() != 2 or table.get_device() != device.index \
            or table.shape[0] != requests:
        raise ValueError(f"block_table must be torch.int64 [{requests}, width] on {device}")
    return table if table.shape[1] <= 1 or table.stride(1) == 1 else table.contiguous()


def _status(status: torch.Tensor | None, device: torch.device) -> int | None:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() != 1 or status.device != device:
        raise ValueError(f"status must be one torch.int32 on {device}")
    return status.data_ptr()


def build_draft_tree(
    parents: torch.Tensor,
    query_start_locations: torch.Tensor,
    committed_lengths: torch.Tensor,
    block_table: torch.Tensor,
    block_size: int,
    *,
    spec=_FULL,
    max_nodes: int = 64,
    status: torch.Tensor | None = None,
) -> DraftTree:
    """Metadata of one draft-tree step, built on the device in one launch.

    ``parents`` int64 [rows]: each node's parent inside its request (an
    earlier node; -1: a root); ``query_start_locations`` int64 [requests + 1];
    ``committed_lengths`` int64 [requests]: tokens already cached;
    ``block_table`` [requests, width] must reach the drafted positions;
    ``spec``: the layer's visibility spec; ``max_nodes``: the most nodes a
    request may have (at most ``MAX_TREE_NODES``).  ``status`` (int32 [1])
    receives the MVB_STATUS_* bits of rows that do not fit."""

    device = parents.device
    if device.type != "cuda":
        raise RuntimeError("b200_paged draft trees require CUDA tensors")
    if not 1 <= max_nodes <= MAX_TREE_NODES:
        raise ValueError(f"max_nodes must be 1 .. {MAX_TREE_NODES}")
    if not 1 <= block_size < 1 << 31:
        raise ValueError("block_size must be positive and fit 32 bits")
    kind, param = spec_code(spec)
    parents = _vector("parents", parents, device)
    committed = _vector("committed_lengths", committed_lengths, device)
    rows, requests, words = parents.shape[0], committed.shape[0], (max_nodes + 63) // 64
    starts = _vector("query_start_locations", query_start_locations, device, requests + 1)
    table = _table(block_table, device, requests)
    buffer = parents.new_empty(rows * (3 + words) + requests)
    positions, context_starts, slots, mask, lengths = buffer.split_with_sizes((rows, rows, rows, rows * words, requests))
    launch(
        _lib.load().mvb_build_draft_tree, device, "b200_paged draft tree",
        parents.data_ptr(), starts.data_ptr(), committed.data_ptr(), table.data_ptr(),
        table.stride(0), table.shape[1], rows, requests, block_size, kind, param, words,
        positions.data_ptr(), context_starts.data_ptr(), lengths.data_ptr(), slots.data_ptr(),
        mask.data_ptr(), _status(status, device),
    )
    return DraftTree(
        AttentionMetadata(
            query_positions=positions, query_context_start_positions=context_starts,
            query_start_locations=starts, context_lengths=lengths, block_table=table,
            slot_mapping=slots, block_size=block_size,
        ),
        mask.view(rows, words),
    )


def accept_draft_tree(
    draft_tokens: torch.Tensor,
    target_tokens: torch.Tensor,
    parents: torch.Tensor,
    query_start_locations: torch.Tensor,
    committed_lengths: torch.Tensor,
    *,
    max_accepted: int,
    status: torch.Tensor | None = None,
) -> AcceptedDraft:
    """The path of each tree that the target keeps, walked on the device.

    ``target_tokens`` int64 [rows] holds the token the target chose at every
    node (``sample_tokens`` over the nodes' logits).  From node 0 (always
    kept) the walk goes to the child drafted with the target's token, the
    first among equals, until there is none or ``max_accepted`` are kept."""

    device = parents.device
    if device.type != "cuda":
        raise RuntimeError("b200_paged draft trees require CUDA tensors")
    if not 1 <= max_accepted <= MAX_TREE_NODES:
        raise ValueError(f"max_accepted must be 1 .. {MAX_TREE_NODES}")
    parents = _vector("parents", parents, device)
    rows = parents.shape[0]
    draft = _vector("draft_tokens", draft_tokens, device, rows)
    target = _vector("target_tokens", target_tokens, device, rows)
    committed = _vector("committed_lengths", committed_lengths, device)
    requests = committed.shape[0]
    starts = _vector("query_start_locations", query_start_locations, device, requests + 1)
    buffer = parents.new_empty(requests * (2 * max_accepted + 3))
    cells = requests * max_accepted
    nodes, tokens, count, lengths, last = buffer.split_with_sizes((cells, cells, requests, requests, requests))
    launch(
        _lib.load().mvb_accept_draft_tree, device, "b200_paged draft acceptance",
        draft.data_ptr(), target.data_ptr(), parents.data_ptr(), starts.data_ptr(), committed.data_ptr(),
        rows, requests, max_accepted, nodes.data_ptr(), count.data_ptr(), tokens.data_ptr(),
        lengths.data_ptr(), last.data_ptr(), _status(status, device),
    )
    return AcceptedDraft(nodes.view(requests, max_accepted), count, tokens.view(requests, max_accepted), lengths, last)


class DraftKVCompactor:
    """Moves the kept nodes' K/V rows behind the committed ones, in place, in
    every layer cache it was made for (one cache group: layers that share a
    block table).  Each cache is a contiguous [2, NB, bs, Hkv, D]; all have
    one shape, dtype and device."""

    __slots__ = ("layer_kv_caches", "_device", "_dtype", "_sizes", "_pointers")

    def __init__(self, layer_kv_caches) -> None:
        caches = tuple(layer_kv_caches)
        if not caches:
            raise ValueError("at least one layer cache is required")
        first = caches[0]
        if first.device.type != "cuda":
            raise RuntimeError("b200_paged draft trees require CUDA tensors")
        if first.dtype not in _CACHE_DTYPES:
            raise ValueError("layer caches must be torch.float16, torch.bfloat16 or torch.float32")
        for t in caches:
            if t.dim() != 5 or t.shape[0] != 2 or not t.is_contiguous():
                raise ValueError("layer caches must be contiguous [2, num_blocks, block_size, num_kv_heads, head_dim]")
            if t.shape != first.shape or t.dtype != first.dtype or t.device != first.device:
                raise ValueError("layer caches must share one shape, dtype and device")
        if first.numel() == 0:
            raise ValueError("layer caches must not be empty")
        begins = sorted(t.data_ptr() for t in caches)
        nbytes = first.numel() * first.element_size()
        if any(b - a < nbytes for a, b in zip(begins, begins[1:])):
            raise ValueError("layer caches must be distinct, without common memory: a row would move twice")
        self.layer_kv_caches = caches
        self._device = first.device
        self._dtype = _CACHE_DTYPES[first.dtype]
        self._sizes = tuple(first.shape[1:])
        self._pointers = ctypes.c_void_p * len(caches)

    def __call__(
        self,
        block_table: torch.Tensor,
        committed_lengths: torch.Tensor,
        nodes: torch.Tensor,
        num_accepted: torch.Tensor,
        *,
        status: torch.Tensor | None = None,
    ) -> None:
        """``committed_lengths``: as before the step; ``nodes`` [requests,
        max_accepted] and ``num_accepted`` as ``accept_draft_tree`` gives
        them.  A request whose nodes do not increase, or whose positions or
        pages are out of range, keeps its rows and sets bits in ``status``."""

        device = self._device
        committed = _vector("committed_lengths", committed_lengths, device)
        requests = committed.shape[0]
        count = _vector("num_accepted", num_accepted, device, requests)
        table = _table(block_table, device, requests)
        if nodes.dtype != torch.int64 or nodes.dim() != 2 or nodes.device != device or nodes.shape[0] != requests:
            raise ValueError(f"nodes must be torch.int64 [{requests}, max_accepted] on {device}")
        if not 1 <= nodes.shape[1] <= MAX_TREE_NODES:
            raise ValueError(f"max_accepted must be 1 .. {MAX_TREE_NODES}")
        if not nodes.is_contiguous():
            nodes = nodes.contiguous()
        blocks, block_size, kv_heads, head_dim = self._sizes
        pointers = self._pointers(*map(torch.Tensor.data_ptr, self.layer_kv_caches))
        launch(
            _lib.load().mvb_compact_draft_kv, device, "b200_paged KV move",
            pointers, len(pointers), blocks, block_size, kv_heads, head_dim, self._dtype,
            table.data_ptr(), table.stride(0), table.shape[1], committed.data_ptr(), nodes.data_ptr(),
            count.data_ptr(), requests, nodes.shape[1], _status(status, device),
        )
