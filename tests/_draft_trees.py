"""Inputs for the draft-tree tests: trees, pages and cached values from a seed."""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch


@dataclass
class TreeBatch:
    parents: torch.Tensor
    starts: torch.Tensor
    committed: torch.Tensor
    table: torch.Tensor
    cache: torch.Tensor
    query: torch.Tensor
    block_size: int

    def to(self, device) -> "TreeBatch":
        moved = {k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in self.__dict__.items()}
        return TreeBatch(**moved)


def make_parents(shape: str, n: int, gen: np.random.Generator) -> list[int]:
    """Parents of n nodes: a chain, a star, two roots, or any earlier node."""

    if shape == "chain":
        return [i - 1 for i in range(n)]
    if shape == "star":
        return [-1] + [0] * (n - 1) if n else []
    if shape == "forest":
        return [-1 if i < 2 else int(gen.integers(0, i)) for i in range(n)]
    return [-1 if i == 0 else int(gen.integers(0, i)) for i in range(n)]


def tree_batch(nodes, committed, *, q_heads=4, kv_heads=2, dim=128, block_size=16, dtype=torch.float16, seed=0,
               shape="any", extra_width=1) -> TreeBatch:
    gen = np.random.default_rng(seed)
    pages = [-(-(c + n) // block_size) for n, c in zip(nodes, committed)]
    blocks = sum(pages) + 2
    order = gen.permutation(blocks)
    table = np.zeros((len(nodes), max([*pages, 0]) + extra_width), np.int64)
    at = 0
    for r, n in enumerate(pages):
        table[r, :n] = order[at: at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int64)
    parents = np.asarray([p for n in nodes for p in make_parents(shape, n, gen)], np.int64)
    normal = torch.Generator().manual_seed(seed)
    rows = int(starts[-1])
    return TreeBatch(
        parents=torch.from_numpy(parents), starts=torch.from_numpy(starts),
        committed=torch.tensor(committed, dtype=torch.int64), table=torch.from_numpy(table),
        cache=torch.randn((2, blocks, block_size, kv_heads, dim), generator=normal).to(dtype),
        query=torch.randn((rows, q_heads, dim), generator=normal).to(dtype), block_size=block_size,
    )


def attention_tolerance(size, reach, exact, dtype, keys: int, dim: int, largest: float) -> np.ndarray:
    """Largest |out - exact| that the roundings allow, per output.

    u = finfo.eps / 2.  The output is rounded once: u(dtype) |exact|.  P is
    rounded to the value's type before P.V: u(dtype) of the weighted |v|
    (``size``); fp32 keeps it.  A score is a sum of dim products in fp32, off by at most
    (dim + 2) 2^-23 times ``reach`` (the largest sum |q||k| scale, tensor
    cores truncating: one whole step per addition), which moves numerator
    and denominator by that factor each; the sums over the keys add keys
    2^-23 each, the exponential and the final division 2^-20."""

    rounded = torch.finfo(dtype).eps / 2
    weight = 0.0 if dtype == torch.float32 else rounded
    score = 2 * (dim + 2) * 2.0 ** -23 * reach[..., None]
    relative = weight + score + 2 * keys * 2.0 ** -23 + 2.0 ** -20
    # Below 2^-14 an fp16 number (a P, or the output) is off by up to 2^-25;
    # the P of a row's largest key is at least 1, so their sum is too.
    floor = 2.0 ** -25 * (1 + keys * largest) if dtype == torch.float16 else 0.0
    return rounded * np.abs(exact) + (1 + rounded) * relative * size + floor + 1e-30
