"""How exact draft-tree attention is, held to what each type's path keeps."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.draft_tree as plain
from _draft_trees import TreeBatch, attention_tolerance, tree_batch
from micro_vllm_b200 import B200PagedAttentionOperator, FullAttentionSpec, build_draft_tree

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
FULL = FullAttentionSpec()


def attend(b, words: int):
    gpu = b.to(DEV)
    tree = build_draft_tree(gpu.parents, gpu.starts, gpu.committed, gpu.table, b.block_size, max_nodes=64 * words)
    out = B200PagedAttentionOperator().attend_tree(gpu.query, gpu.cache, tree)
    _, begin, lengths, _, mask = plain.build_draft_tree(b.parents.numpy(), b.starts.numpy(), b.committed.numpy(),
                                                        b.table.numpy(), b.block_size, FULL.context_start, words)
    exact, size, reach = plain.tree_attention(b.query.float().numpy(), b.cache.float().numpy(), begin, b.starts.numpy(),
                                              lengths, b.table.numpy(), mask, b.query.shape[2] ** -0.5)
    return out.float().cpu().numpy().astype(np.float64), exact, size, reach, int(lengths.max())


@pytest.mark.parametrize("nodes, committed, q_heads, kv_heads", [
    ([8], [257], 16, 8), ([33, 20], [700, 60], 4, 2), ([12, 5], [6000, 900], 16, 2), ([90, 70], [900, 33], 8, 2),
    ([1, 40], [3, 128], 64, 1)])
def test_bf16_weights_keep_sixteen_bits(nodes, committed, q_heads, kv_heads) -> None:
    """As in the paged kernels, a bf16 weight goes through P.V in two parts:
    the first 8 bits, and the rest, below 2^-7 of the weight's power of two,
    rounded to 8 bits: half a step is 2^-16 of the weight.  2^-24 of the weight
    is added to the rest.  fp32's terms are ``attention_tolerance``'s."""

    b = tree_batch(nodes, committed, q_heads=q_heads, kv_heads=kv_heads, dtype=torch.bfloat16, seed=31)
    got, exact, size, reach, keys = attend(b, 2)
    rounded = torch.finfo(torch.bfloat16).eps / 2
    sums = attention_tolerance(size, reach, exact, torch.float32, keys, 128, 0.0)
    allowed = rounded * np.abs(exact) + (1 + rounded) * (sums + (2.0 ** -16 + 2.0 ** -23) * size)
    assert (np.abs(got - exact) <= allowed).all(), (np.abs(got - exact) / allowed).max()


@pytest.mark.parametrize("nodes, q_heads", [(1, 8), (20, 8), (80, 4)])
@pytest.mark.parametrize("bits", [15.5, 21.5, 25.5])
def test_fp16_keeps_the_weights_of_a_long_tail(nodes, q_heads, bits) -> None:
    """Each node's own key outweighs every committed one by 2^bits, and only
    those have a value: what they add up to comes through.  The path scales
    weights so that a row's largest is at least 2^7; below 2^-14 an fp16
    number is off by at most 2^-25, so a weight by 2^-32 of the largest.
    A score is a product of few terms, exact up to its rounding to fp32.  320
    requests over the same pages: items stay whole, long runs of tiles."""

    keys, requests = 4000, 320
    b = tree_batch([nodes], [keys], q_heads=q_heads, kv_heads=1, seed=32, shape="star")
    b.cache.zero_()
    b.query.zero_()
    flat = b.cache.view(2, -1, 1, 128)
    at = lambda p: int(b.table[0, p // 16] * 16 + p % 16)  # noqa: E731
    rise = bits * np.log(2) * 128 ** 0.5 / 16
    for p in range(keys):
        flat[1, at(p)] = 1 + p % 2
    for i in range(nodes):
        flat[0, at(keys + i), 0, i] = 16
        b.query[i, :, i] = rise
    _, exact, size, _, _ = attend(b, 2)
    many = TreeBatch(b.parents.repeat(requests), torch.arange(requests + 1) * nodes, b.committed.repeat(requests),
                     b.table.repeat(requests, 1), b.cache, b.query.repeat(requests, 1, 1), 16).to(DEV)
    tree = build_draft_tree(many.parents, many.starts, many.committed, many.table, 16, max_nodes=128)
    out = B200PagedAttentionOperator().attend_tree(many.query, many.cache, tree)
    got = out.float().cpu().numpy().astype(np.float64).reshape(requests, *exact.shape)
    # Scores: rise in fp16 times 16, scaled in fp32 and cut in ex2 at 2^-20.
    allowed = 2.0 ** -11 * np.abs(exact) + (2.0 ** -11 + 2 * keys * 2.0 ** -23 + 2.0 ** -18) * size
    allowed += 2.0 ** -25 + keys * 2.0 ** -32 * 2
    assert (np.abs(got - exact) <= allowed).all(), (np.abs(got - exact) / allowed).max()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("size", [1, 64, 1024, 2048])
@pytest.mark.parametrize("nodes, committed", [([20], [900]), ([1, 90], [300, 2000])])
def test_large_scores_pick_their_key(nodes, committed, size, dtype) -> None:
    """Queries and keys of +-size: sums of 128 products are exact, scores go
    up to 2^26 in powers of two.  From 64 on, other sums weigh nothing beside a
    row's largest: the output is the mean of the values that have it."""

    b = tree_batch(nodes, committed, q_heads=8, kv_heads=2, dtype=dtype, seed=34)
    b.cache[0] = torch.sign(b.cache[0]) * size
    b.query.copy_(torch.sign(b.query) * size)
    flat = b.cache.view(2, -1, 2, 128)
    for r, c in enumerate(committed):  # a key alike each query of some nodes
        for i in range(0, nodes[r], 7):
            p = (97 * i + 5) % c
            flat[0, int(b.table[r, p // 16] * 16 + p % 16), 0] = b.query[int(b.starts[r]) + i, 1]
    got, exact, weighted, _, keys = attend(b, 2)
    rounded = torch.finfo(dtype).eps / 2
    # The scores' own factor, scale, is rounded to fp32 alike in all of a row's.
    score = 2.0 ** -22 * size * size * 128 ** 0.5 if size == 1 else 0.0
    allowed = 2 * rounded * (np.abs(exact) + weighted) + (score + 2 * keys * 2.0 ** -23 + 2.0 ** -18) * weighted + 2.0 ** -20
    assert np.isfinite(got).all()
    assert (np.abs(got - exact) <= allowed).all(), (np.abs(got - exact) / allowed).max()


def plain_fp32(b, begin, lengths, mask):
    """The attention of one batch in plain fp32 products and sums."""

    out = torch.zeros(b.query.shape)
    group, dim = b.query.shape[1] // b.cache.shape[3], b.query.shape[2]
    words = mask.view(np.uint64)
    for r, length in enumerate(lengths.tolist()):
        first, n = int(b.starts[r]), int(b.starts[r + 1] - b.starts[r])
        at = torch.arange(length)
        k, v = (plane[b.table[r, at // b.block_size], at % b.block_size].repeat_interleave(group, 1) for plane in b.cache)
        seen = torch.zeros(n, length, dtype=torch.bool)
        for i in range(n):
            seen[i, int(begin[first + i]): length - n] = True
            for j in range(n):
                seen[i, length - n + j] = bool((int(words[first + i, j // 64]) >> (j % 64)) & 1)
        score = (b.query[first: first + n].transpose(0, 1) @ k.permute(1, 2, 0)) * dim ** -0.5
        weight = torch.softmax(score.masked_fill(~seen, -torch.inf), 2)
        out[first: first + n] = (weight @ v.transpose(0, 1)).transpose(0, 1)
    return out.numpy().astype(np.float64)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("nodes, committed", [([24, 9], [100, 17]), ([24, 40], [1500, 700]), ([8], [12000])])
def test_fp32_is_as_exact_as_plain_fp32(nodes, committed, dim) -> None:
    """Two parts of 10 and 11 bits keep a factor to 2^-21 (the second is cut
    off: 2^-23 of the factor in the mean square, no sign preferred), so a
    product is off by 2^-22.5 and a sum of ``dim`` of them by sqrt(dim)
    2^-22.5 of a term; plain fp32 rounds every partial sum, dim 2^-25.5 of a
    term for a sequential sum: 8 / sqrt(dim) of it, 1 at 64.  With as much for
    P.V and the sums cut off, twice plain fp32's error in the mean square is
    what the path may have, and as it is spread alike, three times its largest.
    Without the second parts the error is 2^10 times as large."""

    b = tree_batch(nodes, committed, q_heads=4, kv_heads=2, dim=dim, dtype=torch.float32, seed=33)
    got, exact, _, _, _ = attend(b, 1)
    meta = plain.build_draft_tree(b.parents.numpy(), b.starts.numpy(), b.committed.numpy(), b.table.numpy(), b.block_size,
                                  FULL.context_start, 1)
    near = plain_fp32(b, meta[1], meta[2], meta[4])
    rms = lambda x: float(np.sqrt(np.mean(np.square(x - exact))))  # noqa: E731
    assert rms(got) <= 2 * rms(near), (rms(got), rms(near))
    assert np.abs(got - exact).max() <= 3 * np.abs(near - exact).max()
