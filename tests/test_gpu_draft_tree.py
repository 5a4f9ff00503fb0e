"""The draft-tree stages on the GPU against plain loops in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.draft_tree as plain
from _draft_trees import TreeBatch, attention_tolerance, tree_batch
from micro_vllm_b200 import (
    AttentionMetadata,
    B200PagedAttentionOperator,
    ChunkedLocalSpec,
    DraftKVCompactor,
    DraftTree,
    FullAttentionSpec,
    SlidingWindowSpec,
    _lib,
    accept_draft_tree,
    build_draft_tree,
    sample_tokens,
)

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FULL = FullAttentionSpec()


def build(b: TreeBatch, spec=FULL, max_nodes=64, status=None) -> DraftTree:
    return build_draft_tree(b.parents, b.starts, b.committed, b.table, b.block_size, spec=spec, max_nodes=max_nodes,
                            status=status)


def plain_build(b: TreeBatch, spec=FULL, words=1):
    return plain.build_draft_tree(b.parents.numpy(), b.starts.numpy(), b.committed.numpy(), b.table.numpy(),
                                  b.block_size, spec.context_start, words)


def fields(tree: DraftTree):
    md = tree.attention
    return [t.cpu().numpy() for t in (md.query_positions, md.query_context_start_positions, md.context_lengths,
                                      md.slot_mapping, tree.ancestor_mask)]


def check_attention(out: torch.Tensor, b: TreeBatch, meta, *, only=None) -> None:
    """``out`` against the 64-bit loops over the CPU batch ``b``."""

    _, begin, lengths, _, mask = meta
    dim = b.query.shape[2]
    values = b.cache.float().numpy()
    exact, size, reach = plain.tree_attention(b.query.float().numpy(), values, begin, b.starts.numpy(), lengths,
                                              b.table.numpy(), mask, dim ** -0.5)
    finite = np.abs(np.nan_to_num(values[1], nan=0.0, posinf=0.0, neginf=0.0)).max()
    allowed = attention_tolerance(size, reach, exact, out.dtype, int(max(lengths, default=0)), dim, float(finite))
    got = out.float().cpu().numpy().astype(np.float64)
    rows = slice(None) if only is None else only
    np.testing.assert_array_equal(np.isnan(got[rows]), np.isnan(exact[rows]))
    off = np.abs(got[rows] - exact[rows]) - allowed[rows]
    assert np.nanmax(off, initial=-1.0) <= 0, (np.nanmax(off), np.unravel_index(np.nanargmax(off), off.shape))


# ---------------------------------------------------------------- metadata
@pytest.mark.parametrize("shape", ["chain", "star", "forest", "any"])
@pytest.mark.parametrize("spec", [FULL, SlidingWindowSpec(1), SlidingWindowSpec(3), ChunkedLocalSpec(8)])
@pytest.mark.parametrize("max_nodes", [64, 65, 200])
def test_metadata(shape, spec, max_nodes) -> None:
    top = min(max_nodes, 200)
    nodes, committed = [1, 0, top, 7, top - 1, 0], [0, 5, 100, 16, 31, 0]
    b = tree_batch(nodes, committed, q_heads=1, kv_heads=1, dim=8, block_size=16, shape=shape, seed=3)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    words = -(-max_nodes // 64)
    for got, want in zip(fields(build(b.to(DEV), spec, max_nodes, status)), plain_build(b, spec, words)):
        np.testing.assert_array_equal(got, want)
    assert status.item() == 0


def test_metadata_of_the_largest_tree_and_odd_pages() -> None:
    b = tree_batch([1024, 1000], [3, 70], q_heads=1, kv_heads=1, dim=8, block_size=7, shape="chain", seed=4)
    for got, want in zip(fields(build(b.to(DEV), SlidingWindowSpec(130), 1024)), plain_build(b, SlidingWindowSpec(130), 16)):
        np.testing.assert_array_equal(got, want)


def test_metadata_pads_rows_without_an_owner_and_reports_what_does_not_fit() -> None:
    b = tree_batch([3, 4, 2], [5, 9, 20], q_heads=1, kv_heads=1, dim=8)
    b.parents = torch.cat([b.parents, torch.tensor([7, 7, 7])])  # rows behind the last request
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for got, want in zip(fields(build(b.to(DEV), status=status)), plain_build(b)):
        np.testing.assert_array_equal(got, want)
    assert status.item() == 0

    b.parents[1], b.parents[4] = 1, -5  # itself, and no node: both count as roots
    for got, want in zip(fields(build(b.to(DEV), status=status)), plain_build(b)):
        np.testing.assert_array_equal(got, want)
    assert status.item() == _lib.MVB_STATUS_BAD_PARENT
    status.zero_()

    b.committed[2] = 1 << 30  # the second longest length: refused, padded
    for got, want in zip(fields(build(b.to(DEV), status=status)), plain_build(b)):
        np.testing.assert_array_equal(got, want)
    assert status.item() & _lib.MVB_STATUS_INCONSISTENT_COUNTS
    status.zero_()

    short = b.to(DEV)
    short.committed[:] = torch.tensor([5, 60, 0])  # past the second request's table
    tree = build(short, status=status)
    assert tree.attention.slot_mapping[3:7].tolist() == [-1] * 4
    assert status.item() & _lib.MVB_STATUS_POSITION_PAST_TABLE


@pytest.mark.parametrize("starts, owned", [([0, 3, 20, 20], range(0, 3)), ([-2, 3, 7, 9], range(3, 9)),
                                           ([4, 7, 1 << 40, 1 << 40], range(4, 7))], ids=["past", "before", "far"])
def test_metadata_pads_the_rows_of_requests_that_reach_past_them(starts, owned) -> None:
    b = tree_batch([3, 4, 2], [5, 9, 20], q_heads=1, kv_heads=1, dim=8)
    b.parents = torch.cat([torch.full((9,), -1), torch.full((3,), 7)])
    gpu = b.to(DEV)
    gpu.starts = torch.tensor(starts, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    filler = torch.full((12 * 4 + 3,), 1, device=DEV)  # what the allocator may hand out next
    del filler
    positions, begin, _, slots, mask = fields(build(gpu, status=status))
    rest = [t for t in range(12) if t not in owned]
    assert (slots[rest] == -1).all() and not mask[rest].any() and not positions[rest].any() and not begin[rest].any()
    assert (slots[list(owned)] >= 0).all() and mask[list(owned)].all()
    assert status.item() == _lib.MVB_STATUS_INCONSISTENT_COUNTS


def test_metadata_of_lengths_past_the_largest_is_padding() -> None:
    b = tree_batch([3, 4, 2], [5, 9, 20], q_heads=1, kv_heads=1, dim=8)
    gpu = b.to(DEV)
    gpu.committed[:] = torch.tensor([(1 << 63) - 1, -1, -(1 << 63)])
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    positions, _, lengths, slots, mask = fields(build(gpu, status=status))
    assert (slots == -1).all() and not mask.any() and not positions.any() and not lengths.any()
    assert status.item() == _lib.MVB_STATUS_INCONSISTENT_COUNTS


# --------------------------------------------------------------- attention
CASES = [
    # nodes, committed, q_heads, kv_heads, dim, block_size
    ([1], [0], 2, 1, 128, 16),
    ([8], [257], 16, 8, 128, 16),
    ([0, 5, 64, 0, 1, 33, 0], [17, 0, 500, 0, 128, 127, 3], 4, 2, 128, 16),
    ([64, 61], [129, 1], 8, 1, 128, 32),
    ([100, 128], [50, 300], 10, 2, 128, 16),
    ([200], [1000], 6, 2, 128, 64),
    ([3, 17], [250, 6000], 3, 3, 128, 16),
    ([40, 9], [900, 40], 16, 1, 128, 128),
    ([2, 1], [20000, 9], 8, 1, 128, 16),
    ([12, 3], [77, 400], 34, 2, 128, 16),
    ([5], [300], 64, 1, 128, 32),
    ([300, 1], [64, 700], 4, 2, 128, 256),
    ([9, 70], [100, 33], 4, 2, 128, 48),
    ([5, 12], [30, 65], 4, 2, 64, 16),
    ([5, 12], [30, 65], 4, 2, 128, 7),
    ([5, 12], [30, 65], 4, 2, 80, 1),
    ([9, 4], [33, 70], 34, 2, 96, 16),
    ([11], [90], 2, 1, 256, 16),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("case", CASES, ids=[str(i) for i in range(len(CASES))])
def test_attention(case, dtype) -> None:
    nodes, committed, hq, hkv, dim, bs = case
    b = tree_batch(nodes, committed, q_heads=hq, kv_heads=hkv, dim=dim, block_size=bs, dtype=dtype, seed=len(nodes) + hq)
    operator, gpu = B200PagedAttentionOperator(), b.to(DEV)
    out = operator.attend_tree(gpu.query, gpu.cache, build(gpu, max_nodes=300))
    check_attention(out, b, plain_build(b, words=5))
    assert operator.read_status(DEV) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
@pytest.mark.parametrize("spec", [SlidingWindowSpec(1), SlidingWindowSpec(2), SlidingWindowSpec(130),
                                  ChunkedLocalSpec(50), ChunkedLocalSpec(256)])
@pytest.mark.parametrize("shape", ["chain", "forest", "any"])
def test_attention_windows(spec, dtype, shape) -> None:
    b = tree_batch([20, 1, 64, 30], [250, 300, 45, 1021], q_heads=4, kv_heads=2, dtype=dtype, seed=9, shape=shape)
    gpu = b.to(DEV)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, build(gpu, spec))
    check_attention(out, b, plain_build(b, spec))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
def test_attention_of_many_requests_of_mixed_length(dtype) -> None:
    gen = np.random.default_rng(8)
    nodes = gen.integers(0, 20, 450).tolist()
    committed = (2 ** gen.uniform(0, 8.5, 450)).astype(int).tolist()
    b = tree_batch(nodes, committed, q_heads=2, kv_heads=1, dtype=dtype, seed=10)
    gpu = b.to(DEV)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, build(gpu))
    check_attention(out, b, plain_build(b))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_attention_of_more_requests_than_threads(dtype) -> None:
    gen = np.random.default_rng(9)
    nodes, committed = gen.integers(0, 3, 1300).tolist(), gen.integers(0, 25, 1300).tolist()
    nodes[:100] = [0] * 100  # no work where the first threads look
    b = tree_batch(nodes, committed, q_heads=2, kv_heads=2, dtype=dtype, seed=23)
    gpu = b.to(DEV)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, build(gpu))
    check_attention(out, b, plain_build(b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
def test_queries_that_are_not_finite_spoil_their_rows_alone(dtype) -> None:
    b = tree_batch([40, 7], [300, 90], q_heads=4, kv_heads=2, dtype=dtype, seed=24)
    as_bits = torch.int32 if dtype == torch.float32 else torch.int16
    b.query.view(as_bits)[3, 1, 5] = torch.iinfo(as_bits).max  # NaN with every bit of its payload
    b.query[9, 2, 0] = torch.inf
    b.query[44, 0, 127] = -torch.inf
    gpu = b.to(DEV)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, build(gpu))
    for t, h in ((3, 1), (9, 2), (44, 0)):
        assert torch.isnan(out[t, h]).all()
        b.query[t, h], gpu.query[t, h] = 0, 0
        out[t, h] = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, build(gpu))[t, h]
    check_attention(out, b, plain_build(b))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_attention_rows_that_see_nothing_or_have_no_owner_are_zero(dtype) -> None:
    b = tree_batch([4, 3, 2], [0, 20, 40], dtype=dtype, seed=5)
    rows = b.query.shape[0]
    b.query = torch.cat([b.query, torch.ones(3, *b.query.shape[1:], dtype=dtype)])
    b.parents = torch.cat([b.parents, torch.tensor([-1, 0, 1])])
    gpu = b.to(DEV)
    tree = build(gpu)
    mask = tree.ancestor_mask.clone()
    mask[1] = 0  # no committed key, no drafted one
    mask[5] = 0  # committed keys alone
    mask[4] |= 1 << 40  # a bit past the request's nodes
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, DraftTree(tree.attention, mask))
    meta = list(plain_build(b))
    meta[4] = mask.cpu().numpy().copy()
    meta[4][4] &= ~(1 << 40)
    check_attention(out, b, meta)
    assert not out[1].any() and not out[rows:].any() and out[5].any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_attention_of_requests_that_do_not_fit_is_zero(dtype) -> None:
    """More nodes than mask bits, a context shorter than its nodes, rows that
    run backwards or past the batch: zeros there, and the others unharmed."""

    b = tree_batch([70, 5, 4, 6, 3], [40, 50, 60, 200, 70], dtype=dtype, seed=22)
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree = build(gpu, max_nodes=128)
    meta = list(plain_build(b, words=2))
    lengths = tree.attention.context_lengths.clone()
    lengths[2] = 3  # shorter than its 4 nodes
    md = tree.attention
    odd = AttentionMetadata(md.query_positions, md.query_context_start_positions, md.query_start_locations, lengths,
                            md.block_table, md.slot_mapping, 16)
    out = operator.attend_tree(gpu.query, gpu.cache, DraftTree(odd, tree.ancestor_mask[:, :1].contiguous()))
    assert not out[:70].any() and not out[75:79].any()
    rows = [*range(70, 75), *range(79, 88)]
    check_attention(out, b, meta, only=rows)
    starts = md.query_start_locations.clone()
    starts[2], starts[5] = 60, 1000  # request 1 runs backwards, the last one past the rows
    odd = AttentionMetadata(md.query_positions, md.query_context_start_positions, starts, md.context_lengths,
                            md.block_table, md.slot_mapping, 16)
    out = operator.attend_tree(gpu.query, gpu.cache, DraftTree(odd, tree.ancestor_mask))
    torch.cuda.synchronize()
    assert out.shape == gpu.query.shape


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("heads", [(4, 2), (16, 1)])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, heads) -> None:
    """Infinities and NaN in other branches, outside the window and behind
    the last position stay out; in a seen key they come through."""

    b = tree_batch([20, 6], [150, 33], q_heads=heads[0], kv_heads=heads[1], dtype=dtype, seed=6, shape="star")
    spec = SlidingWindowSpec(100)
    flat = b.cache.view(2, -1, heads[1], 128)
    slot = lambda r, p: int(b.table[r, p // 16] * 16 + p % 16)  # noqa: E731
    flat[:, slot(0, 150 + 7)] = torch.nan
    flat[1, slot(0, 150 + 11), :, 3] = torch.inf
    flat[1, slot(0, 150 + 12), :, 5] = -torch.inf
    flat[0, slot(0, 150 + 13)] = torch.inf
    flat[:, slot(0, 40)] = torch.nan  # before every window
    flat[1, slot(0, 51), :, 9] = torch.nan  # the root's window reaches it, its children's do not
    for p in range(33 + 6, 48):
        flat[:, slot(1, p)] = torch.nan  # behind the last node, in its page
    gpu = b.to(DEV)
    tree = build(gpu, spec)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, tree)
    clean = [i for i in range(26) if i not in (0, 7, 11, 12, 13)]
    assert torch.isfinite(out[clean]).all()
    check_attention(out, b, plain_build(b, spec), only=clean)
    assert torch.isnan(out[7]).all()
    assert torch.isnan(out[0, :, 9]).all() and torch.isfinite(out[0, :, :9]).all()
    assert (out[11, :, 3] == torch.inf).all() and torch.isfinite(out[11, :, 4:]).all()
    assert (out[12, :, 5] == -torch.inf).all() and torch.isfinite(out[12, :, :5]).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_attention_hides_missing_pages(dtype) -> None:
    b = tree_batch([7, 5], [200, 64], dtype=dtype, seed=7)
    b.table[0, 3], b.table[0, 7], b.table[1, 0] = -1, 1 << 40, b.cache.shape[1]
    gpu = b.to(DEV)
    operator = B200PagedAttentionOperator()
    out = operator.attend_tree(gpu.query, gpu.cache, build(gpu))
    check_attention(out, b, plain_build(b))
    assert operator.read_status(DEV) == _lib.MVB_STATUS_BLOCK_OUT_OF_RANGE


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32], ids=["fp16", "fp32"])
def test_attention_takes_strides_and_refuses_what_does_not_fit(dtype) -> None:
    b = tree_batch([6, 9], [77, 30], dtype=dtype, seed=11)
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree = build(gpu)
    want = operator.attend_tree(gpu.query, gpu.cache, tree)
    t, h, d = gpu.query.shape
    wide = torch.zeros(t, h + 3, d, dtype=dtype, device=DEV)
    wide[:, 2:2 + h] = gpu.query
    heads_first = gpu.query.transpose(0, 1).contiguous().transpose(0, 1)
    dims_first = gpu.query.transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(t * h * d + 3, dtype=dtype, device=DEV)[3:].view(t, h, d).copy_(gpu.query)
    table = torch.zeros(gpu.table.shape[0], gpu.table.shape[1] + 5, dtype=torch.int64, device=DEV)
    table[:, 2:2 + gpu.table.shape[1]] = gpu.table
    md = tree.attention
    view = AttentionMetadata(md.query_positions, md.query_context_start_positions, md.query_start_locations,
                             md.context_lengths, table[:, 2:2 + gpu.table.shape[1]], md.slot_mapping, 16)
    for query in (wide[:, 2:2 + h], heads_first, dims_first, odd):
        got = operator.attend_tree(query, gpu.cache, DraftTree(view, tree.ancestor_mask))
        check_attention(got, b, plain_build(b))
    two_words = torch.zeros(t, 4, dtype=torch.int64, device=DEV)
    two_words[:, :1] = tree.ancestor_mask
    got = operator.attend_tree(gpu.query, gpu.cache, DraftTree(md, two_words[:, :2]))
    assert torch.equal(got, want)

    with pytest.raises(ValueError, match="multiple"):
        operator.attend_tree(gpu.query[:, :3], gpu.cache, tree)
    with pytest.raises(ValueError, match="dtype"):
        operator.attend_tree(gpu.query.double(), gpu.cache, tree)
    with pytest.raises(ValueError, match="ancestor_mask"):
        operator.attend_tree(gpu.query, gpu.cache, DraftTree(md, tree.ancestor_mask.int()))
    with pytest.raises(ValueError, match="ancestor_mask"):
        operator.attend_tree(gpu.query[1:], gpu.cache, tree)
    with pytest.raises(ValueError, match="contiguous"):
        operator.attend_tree(gpu.query, gpu.cache.transpose(2, 3), tree)
    with pytest.raises(ValueError, match="match"):
        operator.attend_tree(gpu.query, gpu.cache[..., :64].contiguous(), tree)
    empty = operator.attend_tree(gpu.query[:0], gpu.cache, DraftTree(AttentionMetadata(
        md.query_positions[:0], md.query_context_start_positions[:0], torch.zeros(1, dtype=torch.int64, device=DEV),
        md.context_lengths[:0], md.block_table[:0], md.slot_mapping[:0], 16), tree.ancestor_mask[:0]))
    assert empty.shape == (0, h, d)


def test_attention_on_two_streams_and_in_two_graphs() -> None:
    """Calls that overlap, and two captured graphs replayed in turn on new
    inputs, each give what a call alone gives."""

    operator = B200PagedAttentionOperator()
    batches = [tree_batch([16, 30, 9], [2000, 700, 60 + i], q_heads=8, kv_heads=2, dtype=torch.float16, seed=20 + i).to(DEV)
               for i in range(4)]
    trees = [build(b) for b in batches]
    alone = [operator.attend_tree(b.query, b.cache, t) for b, t in zip(batches, trees)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in batches]
    outs: list = [[] for _ in batches]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(operator.attend_tree(batches[i].query, batches[i].cache, trees[i]))
    torch.cuda.synchronize()
    for i, got in enumerate(outs):
        assert all(torch.equal(g, alone[i]) for g in got)

    graphs, results, held = [], [], []
    for i in (0, 1):
        b = batches[i]
        g = torch.cuda.CUDAGraph()
        query = b.query.clone()
        with torch.cuda.graph(g):
            tree = build(b)
            out = operator.attend_tree(query, b.cache, tree)
        graphs.append(g)
        results.append(out)
        held.append((query, tree))
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        assert torch.equal(results[i], alone[i])
    held[0][0].neg_()  # new inputs at the captured addresses
    batches[0].committed.sub_(300)
    graphs[0].replay()
    want = operator.attend_tree(-batches[0].query, batches[0].cache, build(batches[0]))
    torch.cuda.synchronize()
    assert torch.equal(results[0], want)


@pytest.mark.parametrize("dtype, block_size", [(torch.float32, 16), (torch.float16, 48), (torch.bfloat16, 32)],
                         ids=["fp32", "odd-pages", "bf16"])
def test_attention_overlapped_and_replayed_on_other_trees(dtype, block_size) -> None:
    """Calls on three streams at once, and one captured graph replayed on
    lengths, parents and queries that the capture did not see."""

    operator = B200PagedAttentionOperator()
    make = lambda seed, committed: tree_batch([16, 40, 9], committed, q_heads=8, kv_heads=2, dtype=dtype, seed=seed,  # noqa: E731
                                              block_size=block_size)
    b = make(40, [900, 300, 70])
    gpu = b.to(DEV)
    tree = build(gpu)
    want = operator.attend_tree(gpu.query, gpu.cache, tree)
    check_attention(want, b, plain_build(b))
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(20):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(operator.attend_tree(gpu.query, gpu.cache, tree))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = operator.attend_tree(gpu.query, gpu.cache, build(gpu))
    for seed, committed in ((41, [1, 299, 0]), (42, [900, 2, 70])):
        other = make(seed, committed)
        b.parents, b.committed, b.query = other.parents, other.committed, other.query
        for name in ("parents", "committed", "query"):
            getattr(gpu, name).copy_(getattr(b, name))
        graph.replay()
        check_attention(out, b, plain_build(b))


@pytest.mark.parametrize("dtype, code", [(torch.float16, _lib.MVB_DTYPE_F16), (torch.float32, _lib.MVB_DTYPE_F32)],
                         ids=["fp16", "fp32"])
def test_attention_refuses_a_workspace_that_is_missing_or_too_small(dtype, code) -> None:
    b = tree_batch([6, 9], [77, 30], dtype=dtype, seed=11)
    gpu, lib = b.to(DEV), _lib.load()
    tree = build(gpu)
    md, out = tree.attention, torch.full_like(gpu.query, 3)
    rows, q_heads, dim = gpu.query.shape
    _, blocks, block_size, kv_heads, _ = gpu.cache.shape
    need = lib.mvb_tree_attention_workspace_size(rows, 2, q_heads, kv_heads, dim)
    room = torch.empty(need, dtype=torch.uint8, device=DEV)

    def call(workspace, size):
        return lib.mvb_tree_attention(
            gpu.query.data_ptr(), gpu.query.stride(0), gpu.query.stride(1), out.data_ptr(), gpu.cache.data_ptr(),
            blocks, block_size, kv_heads, dim, md.query_context_start_positions.data_ptr(), gpu.starts.data_ptr(),
            md.context_lengths.data_ptr(), gpu.table.data_ptr(), gpu.table.stride(0), gpu.table.shape[1],
            tree.ancestor_mask.data_ptr(), 1, rows, 2, q_heads, dim ** -0.5, code, workspace, size, None,
            torch.cuda.current_stream().cuda_stream)

    assert call(room.data_ptr(), 4096) == _lib.MVB_ERR_WORKSPACE_TOO_SMALL
    assert call(None, need) == _lib.MVB_ERR_INVALID_ARGUMENT
    assert call(room.data_ptr() + 16, need - 16) == _lib.MVB_ERR_INVALID_ARGUMENT
    assert (out == 3).all()
    assert call(room.data_ptr(), need) == _lib.MVB_OK
    check_attention(out, b, plain_build(b))


def test_attention_past_32_bit_offsets() -> None:
    """Pages whose element offset in the cache is past 2^31."""

    blocks = (1 << 31) // (16 * 8 * 128) + 64
    cache = torch.zeros((2, blocks, 16, 8, 128), dtype=torch.float16, device=DEV)
    b = tree_batch([12], [150], q_heads=16, kv_heads=8, seed=12)
    gpu = b.to(DEV)
    pages = b.table.shape[1] - 1
    far = torch.arange(blocks - pages, blocks)
    cache[:, far.to(DEV)] = gpu.cache[:, gpu.table[0, :pages]]
    gpu.table[0, :pages] = far.to(DEV)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, cache, build(gpu))
    check_attention(out, b, plain_build(b))


# -------------------------------------------------------------- acceptance
@pytest.mark.parametrize("shape", ["chain", "star", "forest", "any"])
@pytest.mark.parametrize("most", [1, 3, 16, 300])
def test_acceptance(shape, most) -> None:
    nodes = [1, 0, 2, 64, 17, 300, 0, 1024]
    b = tree_batch(nodes, [4] * 8, q_heads=1, kv_heads=1, dim=8, seed=13, shape=shape)
    gen = np.random.default_rng(most)
    rows = int(b.starts[-1])
    target, draft = gen.integers(0, 3, rows), gen.integers(0, 3, rows)
    for r in range(len(nodes)):  # most drafts agree with their parent's target
        first = int(b.starts[r])
        for i in range(1, nodes[r]):
            if gen.random() < 0.8 and b.parents[first + i] >= 0:
                draft[first + i] = target[first + int(b.parents[first + i])]
    want = plain.accept_draft_tree(draft, target, b.parents.numpy(), b.starts.numpy(), b.committed.numpy(), most)
    gpu, status = b.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    got = accept_draft_tree(torch.from_numpy(draft).to(DEV), torch.from_numpy(target).to(DEV), gpu.parents, gpu.starts,
                            gpu.committed, max_accepted=most, status=status)
    for g, w in zip((got.nodes, got.num_accepted, got.tokens, got.committed_lengths, got.last_rows), want):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    assert status.item() == 0


def test_acceptance_refuses_and_reports() -> None:
    b = tree_batch([4, 3], [5, 6], q_heads=1, kv_heads=1, dim=8).to(DEV)
    zero = torch.zeros(7, dtype=torch.int64, device=DEV)
    args = (b.parents, b.starts, b.committed)
    with pytest.raises(ValueError, match="max_accepted"):
        accept_draft_tree(zero, zero, *args, max_accepted=0)
    with pytest.raises(ValueError, match="draft_tokens"):
        accept_draft_tree(zero[:6], zero, *args, max_accepted=2)
    with pytest.raises(ValueError, match="target_tokens"):
        accept_draft_tree(zero, zero.int(), *args, max_accepted=2)
    with pytest.raises(ValueError, match="query_start_locations"):
        accept_draft_tree(zero, zero, b.parents, b.starts[:2], b.committed, max_accepted=2)
    with pytest.raises(ValueError, match="status"):
        accept_draft_tree(zero, zero, *args, max_accepted=2, status=zero)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    starts = b.starts.clone()
    starts[2] = 9  # past the rows
    got = accept_draft_tree(zero, zero, b.parents, starts, b.committed, max_accepted=2, status=status)
    assert got.num_accepted.tolist() == [2, 0] and got.last_rows.tolist()[1] == -1
    assert got.nodes[1].tolist() == [-1, -1] and got.committed_lengths.tolist() == [7, 6]
    assert status.item() == _lib.MVB_STATUS_INCONSISTENT_COUNTS
    none = accept_draft_tree(zero[:0], zero[:0], b.parents[:0], b.starts[:1], b.committed[:0], max_accepted=2)
    assert none.nodes.shape == (0, 2)


# ----------------------------------------------------------------- KV move
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("kv_heads, dim, block_size", [(8, 128, 16), (2, 64, 7), (1, 5, 1), (3, 96, 32)])
@pytest.mark.parametrize("layers", [1, 3, 70])
def test_kv_move(dtype, kv_heads, dim, block_size, layers) -> None:
    gen = np.random.default_rng(layers)
    nodes, committed = [20, 1, 0, 64, 33], [0, 5, 6, 31, 100]
    b = tree_batch(nodes, committed, q_heads=kv_heads, kv_heads=kv_heads, dim=dim, block_size=block_size, seed=14)
    most = 40
    path, count = np.full((5, most), -1, np.int64), np.zeros(5, np.int64)
    for r, n in enumerate(nodes):
        keep = sorted({0, *gen.integers(0, n, 1 + n // 2).tolist()})[:most] if n else []
        if r == 3:
            keep = list(range(24, 64))  # every source but the last ones is a target too
        path[r, :len(keep)], count[r] = keep, len(keep)
    normal = torch.Generator(device=DEV).manual_seed(layers)
    caches = [torch.randn(b.cache.shape, generator=normal, device=DEV).to(dtype) for _ in range(layers)]
    caches[0].view(-1)[:9] = torch.nan
    as_bits = torch.int32 if dtype == torch.float32 else torch.int16
    want = [plain.compact_draft_kv(c.view(as_bits).cpu().numpy(), b.table.numpy(), b.committed.numpy(), path, count)
            for c in caches]
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    gpu = b.to(DEV)
    DraftKVCompactor(caches)(gpu.table, gpu.committed, torch.from_numpy(path).to(DEV), torch.from_numpy(count).to(DEV),
                             status=status)
    for c, w in zip(caches, want):
        np.testing.assert_array_equal(c.view(as_bits).cpu().numpy(), w)
    assert status.item() == 0


def test_kv_move_leaves_requests_that_do_not_fit() -> None:
    b = tree_batch([8, 8, 8, 8, 8, 8], [20] * 6, kv_heads=1, dim=8, seed=15)
    gpu = b.to(DEV)
    path = torch.tensor([[0, 2, 5], [0, 5, 2], [0, 2, 900], [0, 3, 4], [0, 1, 7], [-1, 2, 3]], device=DEV)
    count = torch.tensor([3, 3, 3, 4, 3, 2], device=DEV)
    gpu.table[4, 1] = 77  # no such block: holds positions 20 .. 27
    before, status = gpu.cache.clone(), torch.zeros(1, dtype=torch.int32, device=DEV)
    DraftKVCompactor([gpu.cache])(gpu.table, gpu.committed, path, count, status=status)
    want = plain.compact_draft_kv(before.view(torch.int16).cpu().numpy(), b.table.numpy(), np.array([20]), path[:1].cpu().numpy(),
                                  np.array([3]))
    np.testing.assert_array_equal(gpu.cache.view(torch.int16).cpu().numpy(), want)
    assert status.item() == (_lib.MVB_STATUS_INCONSISTENT_COUNTS | _lib.MVB_STATUS_POSITION_PAST_TABLE
                             | _lib.MVB_STATUS_BLOCK_OUT_OF_RANGE)
    move = DraftKVCompactor([gpu.cache])
    with pytest.raises(ValueError, match="num_accepted"):
        move(gpu.table, gpu.committed, path, count[:5])
    with pytest.raises(ValueError, match="nodes"):
        move(gpu.table, gpu.committed, path.int(), count)
    with pytest.raises(ValueError, match="max_accepted"):
        move(gpu.table, gpu.committed, path[:, :0], count)
    with pytest.raises(ValueError, match="share one shape"):
        DraftKVCompactor([gpu.cache, gpu.cache.float()])
    with pytest.raises(ValueError, match="contiguous"):
        DraftKVCompactor([gpu.cache[:, ::2]])
    with pytest.raises(ValueError, match="distinct"):
        DraftKVCompactor([gpu.cache, gpu.cache])


# --------------------------------------------------------- steps in a row
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_steps_in_a_row(captured) -> None:
    """Four steps as a serving loop runs them (write, attend, sample, accept,
    move), eager and as one captured graph, against the 64-bit loops: every
    step's attention, and the cache that the kept tokens leave."""

    layers, most, vocab, steps = 2, 6, 11, 4
    nodes, committed = [12, 1, 30], [40, 3, 130]
    room = [c + n + steps * most for n, c in zip(nodes, committed)]
    b = tree_batch(nodes, room, q_heads=4, kv_heads=2, dtype=torch.float16, seed=16)
    b.committed = torch.tensor(committed)
    normal = torch.Generator().manual_seed(17)
    rows = b.query.shape[0]
    keys, values, queries = (torch.randn((steps, layers, rows, h, 128), generator=normal).to(torch.float16) for h in (2, 2, 4))
    drafts = torch.randint(0, vocab, (steps, rows), generator=normal)
    logits = torch.randn((steps, rows, vocab), generator=normal)
    caches = [b.cache.clone() for _ in range(layers)]
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    live = [c.to(DEV) for c in caches]
    move = DraftKVCompactor(live)
    k, v, q, lg, dr = (t[0].to(DEV) for t in (keys, values, queries, logits, drafts))
    greedy = (torch.zeros(rows, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV), torch.ones(rows, device=DEV),
              torch.zeros(rows, dtype=torch.int64, device=DEV), torch.zeros(rows, dtype=torch.int64, device=DEV))
    length = gpu.committed.clone()

    def step():
        tree = build_draft_tree(gpu.parents, gpu.starts, length, gpu.table, 16)
        outs = [operator.forward_tree(q[i], k[i], v[i], live[i], tree) for i in range(layers)]
        kept = accept_draft_tree(dr, sample_tokens(lg, *greedy), gpu.parents, gpu.starts, length, max_accepted=most)
        move(gpu.table, length, kept.nodes, kept.num_accepted)
        length.copy_(kept.committed_lengths)
        return outs, kept

    graph = None
    if captured:
        saved = [c.clone() for c in live]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs, kept = step()
        for c, s in zip(live, saved):
            c.copy_(s)
        length.copy_(gpu.committed)
    for n in range(steps):
        for dst, src in ((k, keys), (v, values), (q, queries), (lg, logits), (dr, drafts)):
            dst.copy_(src[n])
        if captured:
            graph.replay()
        else:
            outs, kept = step()
        meta = plain_build(b)
        target = logits[n].argmax(1).numpy()
        want = plain.accept_draft_tree(drafts[n].numpy(), target, b.parents.numpy(), b.starts.numpy(), b.committed.numpy(), most)
        for i in range(layers):
            flat = caches[i].view(2, -1, 2, 128)
            flat[0, torch.from_numpy(meta[3])], flat[1, torch.from_numpy(meta[3])] = keys[n, i], values[n, i]
            b.cache, b.query = caches[i], queries[n, i]
            check_attention(outs[i], b, meta)
            moved = plain.compact_draft_kv(caches[i].view(torch.int16).numpy(), b.table.numpy(), b.committed.numpy(), want[0], want[1])
            caches[i] = torch.from_numpy(moved).view(torch.float16)
            assert torch.equal(live[i].cpu().view(torch.int16), caches[i].view(torch.int16))
        for got, w in zip((kept.nodes, kept.num_accepted, kept.tokens, kept.committed_lengths, kept.last_rows), want):
            np.testing.assert_array_equal(got.cpu().numpy(), w)
        b.committed = torch.from_numpy(want[3])


def test_a_chain_of_drafts_equals_paged_attention() -> None:
    """A chain is a causal chunk: the framework's own paged attention gives
    the same rows, to the tolerance of both."""

    b = tree_batch([7, 30], [300, 90], q_heads=4, kv_heads=2, dtype=torch.float16, seed=18, shape="chain")
    gpu, operator = b.to(DEV), B200PagedAttentionOperator()
    tree = build(gpu)
    check_attention(operator.attend(gpu.query, gpu.cache, tree.attention), b, plain_build(b))
    check_attention(operator.attend_tree(gpu.query, gpu.cache, tree), b, plain_build(b))
