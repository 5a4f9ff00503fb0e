"""Draft trees where one mechanism meets another: values that are not finite
in items of many tiles, first calls inside a capture, windows with missing
pages, far offsets, the layer's prologue, several cache groups."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.draft_tree as plain
from _draft_trees import attention_tolerance, tree_batch
from micro_vllm_b200 import (
    B200PagedAttentionOperator,
    ChunkedLocalSpec,
    DraftTree,
    AttentionMetadata,
    FullAttentionSpec,
    SlidingWindowSpec,
    _lib,
    build_draft_tree,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FULL = FullAttentionSpec()
DTYPES = pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])


def build(b, spec=FULL, max_nodes=64):
    return build_draft_tree(b.parents, b.starts, b.committed, b.table, b.block_size, spec=spec, max_nodes=max_nodes)


def plain_build(b, spec=FULL, words=1):
    return plain.build_draft_tree(b.parents.numpy(), b.starts.numpy(), b.committed.numpy(), b.table.numpy(),
                                  b.block_size, spec.context_start, words)


def check(out, b, meta, *, only=slice(None)) -> None:
    """``out`` against the 64-bit loops, infinities and NaN among it."""

    _, begin, lengths, _, mask = meta
    dim, values = b.query.shape[2], b.cache.float().numpy()
    with np.errstate(all="ignore"):
        exact, size, reach = plain.tree_attention(b.query.float().numpy(), values, begin, b.starts.numpy(), lengths,
                                                  b.table.numpy(), mask, dim ** -0.5)
    finite = np.abs(np.nan_to_num(values[1], nan=0.0, posinf=0.0, neginf=0.0)).max()
    allowed = attention_tolerance(size, reach, exact, out.dtype, int(max(lengths)), dim, float(finite))[only]
    got, exact = out.float().cpu().numpy().astype(np.float64)[only], exact[only]
    np.testing.assert_array_equal(np.isnan(got), np.isnan(exact))
    odd = ~np.isfinite(exact)
    np.testing.assert_array_equal(got[odd], exact[odd])
    assert np.isfinite(got[~odd]).all()
    assert (np.abs(got[~odd] - exact[~odd]) <= allowed[~odd]).all()


def spoil(b, r: int, position: int, value: float, *, plane=1, column=slice(None), head=slice(None)) -> None:
    page = int(b.table[r, position // b.block_size])
    b.cache[plane, page, position % b.block_size, head, column] = value


def on_tensor_tiles(query, out, cache) -> int:
    rows, q_heads, dim = query.shape
    _, blocks, block_size, kv_heads, _ = cache.shape
    code = {torch.float16: _lib.MVB_DTYPE_F16, torch.bfloat16: _lib.MVB_DTYPE_BF16, torch.float32: _lib.MVB_DTYPE_F32}
    return _lib.load().mvb_tree_attention_uses_tcgen05(
        query.data_ptr(), query.stride(0), query.stride(1), out.data_ptr(), cache.data_ptr(), blocks, block_size,
        kv_heads, dim, rows, 4, q_heads, code[query.dtype])


@DTYPES
def test_which_kernel_runs(dtype) -> None:
    """The 16-bit tests of the tensor tiles run on them: a build whose
    register count does not fit the kernel's split would fail here."""

    def path(q_heads=16, kv_heads=8, dim=128, block_size=16, rows=24, cut=0):
        query = torch.zeros(rows * (q_heads * dim + cut) + cut, dtype=dtype, device=DEV)
        query = query[cut:].view(rows, -1)[:, :q_heads * dim].view(rows, q_heads, dim)
        cache = torch.zeros(2, 5, block_size, kv_heads, dim, dtype=dtype, device=DEV)
        return on_tensor_tiles(query, torch.empty_like(query), cache)

    tiles = int(dtype != torch.float32)
    for block_size in (16, 32, 64, 128, 256, 512):
        assert path(block_size=block_size) == tiles
    for q_heads, kv_heads in ((1, 1), (8, 8), (6, 2), (10, 2), (32, 8), (64, 1)):
        assert path(q_heads, kv_heads) == path(q_heads, kv_heads, rows=1) == tiles
    assert path(cut=8) == tiles
    # Just outside: pages of no power of two or below 16, wider groups, other
    # head sizes, rows that are not 16-byte aligned.
    assert path(block_size=48) == path(block_size=8) == path(130, 2) == path(dim=64) == path(dim=136) == path(cut=4) == 0


def test_slots_of_pages_that_cannot_be_do_not_wrap() -> None:
    """16 times 2^60 is 0 in 64 bits: a node on such a page has no slot."""

    b = tree_batch([3, 2], [14, 30], q_heads=1, kv_heads=1, dim=8)
    want = plain_build(b)[3].tolist()
    b.table[0, 1], b.table[1, 1] = 1 << 60, (1 << 63) - 1
    gpu = b.to(DEV)
    slots = build(gpu).attention.slot_mapping.tolist()
    assert slots == [want[0], want[1], -1, -1, -1]
    gpu.table[1, 1] = (1 << 32) - 1
    assert build(gpu).attention.slot_mapping.tolist()[3] == ((1 << 32) - 1) * 16 + 14


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_a_status_word_keeps_its_bits_over_captured_calls(dtype) -> None:
    """An operator whose first call is captured: nothing is set before the
    graph runs, and a replay or a call that is clean clears nothing."""

    b = tree_batch([7, 5], [200, 64], dtype=dtype, seed=55)
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree = build(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = operator.attend_tree(gpu.query, gpu.cache, tree)
    assert operator.read_status(DEV) == 0
    whole = gpu.table.clone()
    gpu.table[0, 3] = -1
    graph.replay()
    gpu.table.copy_(whole)
    graph.replay()
    operator.attend_tree(gpu.query, gpu.cache, tree)
    assert operator.read_status(DEV) == _lib.MVB_STATUS_BLOCK_OUT_OF_RANGE
    assert operator.read_status(DEV) == 0
    check(out, b, plain_build(b))
    late = B200PagedAttentionOperator()
    late._devices.clear()  # as one made before CUDA is in use, or for another device
    with pytest.raises(RuntimeError, match="no status word"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            late.attend_tree(gpu.query, gpu.cache, tree)
    assert not late._devices
    assert late.read_status(DEV) == 0 and torch.equal(late.attend_tree(gpu.query, gpu.cache, tree), out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_forward_tree_refuses_before_it_writes(dtype) -> None:
    b = tree_batch([6, 9], [77, 30], dtype=dtype, seed=56)
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree = build(gpu)
    md, rows = tree.attention, b.query.shape[0]
    key = torch.ones(rows, 2, 128, dtype=dtype, device=DEV)

    def refused(match, *, mask=tree.ancestor_mask, query=gpu.query, key=key, **fields):
        other = AttentionMetadata(**{**{f: getattr(md, f) for f in md.__dataclass_fields__}, **fields})
        with pytest.raises(ValueError, match=match):
            operator.forward_tree(query, key, key, gpu.cache, DraftTree(other, mask))

    for slots in (md.slot_mapping[:-1], torch.cat([md.slot_mapping, md.slot_mapping]), md.slot_mapping.int(),
                  md.slot_mapping.cpu(), md.slot_mapping[:0]):
        refused("slot_mapping", slot_mapping=slots)
    refused("block_table", block_table=md.block_table[:1])
    refused("match the query", query_start_locations=md.query_start_locations[:-1])
    refused("match the query", query_context_start_positions=md.query_context_start_positions[1:])
    refused("context_lengths", context_lengths=md.context_lengths.int())
    refused("ancestor_mask", mask=tree.ancestor_mask[1:])
    refused("key/value", key=key[1:])
    refused("multiple", query=gpu.query[:, :0])
    assert torch.equal(gpu.cache.cpu(), b.cache)
    wide = torch.zeros(2, 4, 16, 2, 264, dtype=dtype, device=DEV)
    with pytest.raises(ValueError, match="head_dim"):
        operator.attend_tree(wide.new_zeros(rows, 4, 264), wide, tree)
    with pytest.raises(ValueError, match="head_dim"):
        operator.attend_tree(gpu.query[..., :0], wide[..., :0].contiguous(), tree)
