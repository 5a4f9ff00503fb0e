"""How exact draft-tree attention is, held to what each type's path keeps."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import oracle.draft_tree as plain
from _draft_trees import attention_tolerance, tree_batch
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
