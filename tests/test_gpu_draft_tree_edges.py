"""Draft trees where one mechanism meets another: values that are not finite
in items of many tiles, first calls inside a capture, windows with missing
pages, far offsets, the layer's prologue, several cache groups."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.draft_tree as plain
from _draft_trees import attention_tolerance, tree_batch
from _golden import within_ulps
from micro_vllm_b200 import (
    AttentionMetadata,
    B200PagedAttentionOperator,
    ChunkedLocalSpec,
    DraftKVCompactor,
    DraftTree,
    FullAttentionSpec,
    Qwen3AttentionPrologue,
    SlidingWindowSpec,
    _lib,
    accept_draft_tree,
    build_draft_tree,
    rotary_inverse_frequencies,
)
from oracle.qk_prologue import qk_norm_rope_and_cache

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


def test_many_operators_are_first_called_in_one_capture() -> None:
    """More of them than torch has streams, the captured one among these."""

    b = tree_batch([7], [40], seed=55)
    gpu = b.to(DEV)
    tree = build(gpu)
    want = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, tree)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        operators = [B200PagedAttentionOperator() for _ in range(70)]
        outs = [operator.attend_tree(gpu.query, gpu.cache, tree) for operator in operators]
    graph.replay()
    assert all(torch.equal(out, want) for out in outs)
    assert [operator.read_status(DEV) for operator in operators] == [0] * 70


@pytest.mark.parametrize("inside", [True, False])
def test_the_status_is_read_in_and_out_of_inference_mode(inside) -> None:
    b = tree_batch([7, 5], [200, 64], seed=55)
    b.table[0, 3] = -1
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    with torch.inference_mode(inside):
        operator.attend_tree(gpu.query, gpu.cache, build(gpu))
    with torch.inference_mode(not inside):
        assert operator.read_status(DEV) == _lib.MVB_STATUS_BLOCK_OUT_OF_RANGE
    assert operator.read_status(DEV) == 0


def test_metadata_refuses_sizes_that_do_not_fit() -> None:
    gpu = tree_batch([3, 2], [14, 30], q_heads=1, kv_heads=1, dim=8).to(DEV)
    for block_size in (0, -16, 1 << 31, (1 << 32) + 16):  # the last is 16 in 32 bits
        with pytest.raises(ValueError, match="block_size"):
            build_draft_tree(gpu.parents, gpu.starts, gpu.committed, gpu.table, block_size)
    for max_nodes in (0, -1, 1025, (1 << 32) + 64):
        with pytest.raises(ValueError, match="max_nodes"):
            build_draft_tree(gpu.parents, gpu.starts, gpu.committed, gpu.table, 16, max_nodes=max_nodes)


def test_kv_move_refuses_caches_that_overlap() -> None:
    flat = torch.zeros(3 * 2 * 4 * 16 * 2 * 8, dtype=torch.float16, device=DEV)
    size = flat.numel() // 3
    cut = lambda at: flat[at: at + size].view(2, 4, 16, 2, 8)  # noqa: E731
    DraftKVCompactor([cut(2 * size), cut(0), cut(size)])
    for at in (0, 8, size // 2, size - 8):
        with pytest.raises(ValueError, match="distinct"):
            DraftKVCompactor([cut(2 * size), cut(0), cut(at)])


# Requests x heads against the GPU's CTAs: a few long requests are cut into
# shares of a tile or two, many middling ones leave whole items of several tiles.
FEW = ([40, 7, 150, 0, 260], [3000, 901, 1290, 77, 2000])
MANY = ([5, 12, 3, 9] * 12, [700, 391, 600, 515] * 12)


@DTYPES
@pytest.mark.parametrize("heads", [(4, 2), (16, 8)], ids=["4x2", "16x8"])
@pytest.mark.parametrize("sizes", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("spec", [FULL, SlidingWindowSpec(333)], ids=["full", "window"])
def test_values_that_are_not_finite_in_items_of_many_tiles(sizes, heads, spec, dtype) -> None:
    nodes, committed = sizes
    b = tree_batch(nodes, committed, q_heads=heads[0], kv_heads=heads[1], dtype=dtype, seed=51)
    gen = np.random.default_rng(52)
    bad = [torch.nan, torch.inf, -torch.inf]
    for r, (n, c) in enumerate(zip(nodes, committed)):
        if n == 0 or r % 4 == 3:
            continue  # some requests stay clean
        for i in range(0, n, 3):  # drafted branches, in every one of their tiles
            if gen.random() < 0.4:
                spoil(b, r, c + i, bad[i % 3], column=int(gen.integers(0, 128)), head=int(gen.integers(0, heads[1])))
        if spec is not FULL:
            for d in range(6):  # the window's edge: seen by the nodes near the root
                spoil(b, r, c - 333 + 1 + d, bad[d % 3], column=5 * d)
            spoil(b, r, c - 334, torch.nan)  # seen by none
            spoil(b, r, c - 334, torch.nan, plane=0)
        for p in range(c + n, -(-(c + n) // 16) * 16):  # behind the last node
            spoil(b, r, p, torch.nan)
            spoil(b, r, p, torch.nan, plane=0)
    gpu = b.to(DEV)
    operator = B200PagedAttentionOperator()
    out = operator.attend_tree(gpu.query, gpu.cache, build(gpu, spec, 320))
    check(out, b, plain_build(b, spec, 5))
    assert operator.read_status(DEV) == 0


@DTYPES
@pytest.mark.parametrize("sizes", [FEW, MANY], ids=["few", "many"])
def test_infinite_values_that_every_row_sees(sizes, dtype) -> None:
    nodes, committed = sizes
    b = tree_batch(nodes, committed, q_heads=4, kv_heads=2, dtype=dtype, seed=53)
    for r, c in enumerate(committed):
        spoil(b, r, c // 2, torch.inf, column=3)
        spoil(b, r, c // 3, -torch.inf, column=9, head=1)
        spoil(b, r, c // 5, torch.nan, column=100)
    gpu = b.to(DEV)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, build(gpu, max_nodes=320))
    check(out, b, plain_build(b, words=5))


@DTYPES
@pytest.mark.parametrize("spec", [SlidingWindowSpec(1), SlidingWindowSpec(130), ChunkedLocalSpec(256)])
def test_windows_with_missing_pages(spec, dtype) -> None:
    b = tree_batch([20, 1, 64, 30], [250, 300, 45, 1021], q_heads=4, kv_heads=2, dtype=dtype, seed=54)
    b.table[0, 13], b.table[0, 15], b.table[3, 60], b.table[3, 61] = -1, 1 << 40, b.cache.shape[1], -5
    gpu = b.to(DEV)
    operator = B200PagedAttentionOperator()
    out = operator.attend_tree(gpu.query, gpu.cache, build(gpu, spec))
    check(out, b, plain_build(b, spec))
    assert operator.read_status(DEV) == _lib.MVB_STATUS_BLOCK_OUT_OF_RANGE


@DTYPES
def test_requests_that_run_backwards_leave_the_others_unharmed(dtype) -> None:
    """Rows that two requests claim are undefined; all others are theirs."""

    b = tree_batch([70, 5, 4, 6, 3], [40, 50, 60, 200, 70], dtype=dtype, seed=22)
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree = build(gpu, max_nodes=128)
    md = tree.attention
    starts = md.query_start_locations.clone()
    starts[2], starts[5] = 60, 1000  # request 1 runs backwards, the last one past the rows
    odd = AttentionMetadata(md.query_positions, md.query_context_start_positions, starts, md.context_lengths,
                            md.block_table, md.slot_mapping, 16)
    out = operator.attend_tree(gpu.query, gpu.cache, DraftTree(odd, tree.ancestor_mask))
    check(out, b, plain_build(b, words=2), only=[*range(60), *range(79, 85)])
    assert not out[85:].any()


@pytest.mark.parametrize("made", ["before", "in-capture"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_a_status_word_keeps_its_bits_over_captured_calls(dtype, made) -> None:
    """An operator whose first call is captured: nothing is set before the
    graph runs, and a replay or a call that is clean clears nothing."""

    b = tree_batch([7, 5], [200, 64], dtype=dtype, seed=55)
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree = build(gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        scratch = gpu.query * 3  # memory of the graph's own pool, free again
        del scratch
        if made == "in-capture":
            operator = B200PagedAttentionOperator()
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


@pytest.mark.parametrize("block_size", [16, 48], ids=["pages", "odd-pages"])
def test_attention_past_32_bit_offsets_off_the_tensor_tiles(block_size) -> None:
    """fp32, and 16 bits with pages that are no power of two, at element
    offsets past 2^31."""

    dtype = torch.float32 if block_size == 16 else torch.bfloat16
    blocks = (1 << 31) // (block_size * 8 * 128) + 64
    b = tree_batch([12], [150], q_heads=16, kv_heads=8, seed=12, dtype=dtype, block_size=block_size)
    cache = torch.zeros((2, blocks, block_size, 8, 128), dtype=dtype, device=DEV)
    gpu = b.to(DEV)
    pages = b.table.shape[1] - 1
    far = torch.arange(blocks - pages, blocks, device=DEV)
    cache[:, far] = gpu.cache[:, gpu.table[0, :pages]]
    gpu.table[0, :pages] = far
    check(B200PagedAttentionOperator().attend_tree(gpu.query, cache, build(gpu)), b, plain_build(b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("spec", [FULL, SlidingWindowSpec(20)], ids=["full", "window"])
def test_a_layer_through_the_prologue(spec, dtype) -> None:
    """Projections, the fused prologue with the tree's metadata, attend_tree:
    siblings share a rotary position and no slot."""

    name = {torch.float16: "f16", torch.bfloat16: "bf16"}[dtype]
    b = tree_batch([12, 1, 0, 30], [40, 3, 9, 130], q_heads=16, kv_heads=8, dtype=dtype, seed=57)
    rows, normal = b.query.shape[0], torch.Generator().manual_seed(58)
    fused = (torch.randn((rows, 32 * 128), generator=normal) * 2).to(dtype).to(DEV)
    q, k, v = (part.unflatten(1, (-1, 128)) for part in fused.split([16 * 128, 8 * 128, 8 * 128], 1))
    weights = (0.5 + torch.rand(2, 128, generator=normal)).to(dtype).to(DEV)
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree, meta = build(gpu, spec), plain_build(b, spec)
    md = tree.attention
    prologue = Qwen3AttentionPrologue(weights[0], weights[1], 1e-6, 1e6)
    rotated = prologue(md.query_positions, q, k, v, gpu.cache, md)
    out = operator.attend_tree(rotated, gpu.cache, tree)

    want_cache = b.cache.float().numpy().copy()
    inverse = rotary_inverse_frequencies(128, 1e6, DEV).cpu().numpy()
    want_q = qk_norm_rope_and_cache(
        *(t.float().cpu().numpy() for t in (q, k, v)), meta[0], weights[0].float().cpu().numpy(),
        weights[1].float().cpu().numpy(), 1e-6, inverse, want_cache, meta[3], name)
    got_cache = gpu.cache.float().cpu().numpy()
    assert within_ulps(rotated.float().cpu().numpy(), want_q, name, 2, rotated=True).all()
    assert within_ulps(got_cache[0], want_cache[0], name, 2, rotated=True).all()
    np.testing.assert_array_equal(got_cache[1], want_cache[1])
    b.query, b.cache = rotated.cpu(), gpu.cache.cpu()
    check(out, b, meta)


@DTYPES
def test_two_cache_groups_in_one_step(dtype) -> None:
    """Layers of full attention and layers of a sliding window keep tables,
    trees and moves of their own; the accepted path is one."""

    nodes, committed, most = [12, 1, 30], [40, 3, 130], 6
    room = [c + n for c, n in zip(committed, nodes)]
    specs = [FULL, SlidingWindowSpec(25)]
    groups = [tree_batch(nodes, room, q_heads=4, kv_heads=2, dtype=dtype, seed=60 + i) for i in range(2)]
    for b in groups:
        b.committed, b.parents = torch.tensor(committed), groups[0].parents
    rows, normal = groups[0].query.shape[0], torch.Generator().manual_seed(62)
    target = torch.randint(0, 4, (rows,), generator=normal)
    drafts = torch.randint(0, 4, (rows,), generator=normal)
    on_gpu = [b.to(DEV) for b in groups]
    operator = B200PagedAttentionOperator()
    keys, values = (torch.randn((2, rows, 2, 128), generator=normal).to(dtype) for _ in range(2))
    outs = [operator.forward_tree(g.query, k.to(DEV), v.to(DEV), g.cache, build(g, spec))
            for g, spec, k, v in zip(on_gpu, specs, keys, values)]
    first = on_gpu[0]
    kept = accept_draft_tree(drafts.to(DEV), target.to(DEV), first.parents, first.starts, first.committed, max_accepted=most)
    for g in on_gpu:
        DraftKVCompactor([g.cache])(g.table, g.committed, kept.nodes, kept.num_accepted)
    want = plain.accept_draft_tree(drafts.numpy(), target.numpy(), groups[0].parents.numpy(), groups[0].starts.numpy(),
                                   groups[0].committed.numpy(), most)
    np.testing.assert_array_equal(kept.nodes.cpu().numpy(), want[0])
    bits = torch.int32 if dtype == torch.float32 else torch.int16
    for b, g, spec, out, k, v in zip(groups, on_gpu, specs, outs, keys, values):
        meta = plain_build(b, spec)
        flat = b.cache.view(2, -1, 2, 128)
        flat[0, torch.from_numpy(meta[3])], flat[1, torch.from_numpy(meta[3])] = k, v
        check(out, b, meta)
        moved = plain.compact_draft_kv(b.cache.view(bits).numpy(), b.table.numpy(), b.committed.numpy(), want[0], want[1])
        np.testing.assert_array_equal(g.cache.view(bits).cpu().numpy(), moved)
        for r, c in enumerate(committed):  # a kept node lies where its rotary position says
            path = want[0][r, :want[1][r]]
            np.testing.assert_array_equal(meta[0][int(b.starts[r]) + path], c + np.arange(len(path)))
