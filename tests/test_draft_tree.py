"""Draft trees on the CPU: the oracle's known answers, and what the entry
points refuse before anything runs on a device."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import oracle.draft_tree as plain
from _draft_trees import tree_batch
from micro_vllm_b200 import (
    AttentionMetadata,
    B200PagedAttentionOperator,
    DraftKVCompactor,
    DraftTree,
    _lib,
    accept_draft_tree,
    build_draft_tree,
)
from micro_vllm_b200.build import build

FAKE = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib() -> ctypes.CDLL:
    build()
    return _lib.load()


def full(position: int) -> int:
    return 0


def test_metadata_of_a_known_tree() -> None:
    #      0          request 0 of two, 3 committed tokens; request 1 drafts
    #    1   2        nothing; pages of 4 tokens.
    #        3
    parents, starts = np.array([-1, 0, 0, 2]), np.array([0, 4, 4])
    table = np.array([[5, 7], [1, 1]])
    got = plain.build_draft_tree(parents, starts, np.array([3, 6]), table, 4, full, 1)
    positions, begin, lengths, slots, mask = (g.tolist() for g in got)
    assert positions == [3, 4, 4, 5]
    assert begin == [0, 0, 0, 0]
    assert lengths == [7, 6]
    assert slots == [23, 28, 29, 30]
    assert mask == [[0b1], [0b11], [0b101], [0b1101]]
    # A window of two tokens: each node sees itself and its parent.
    got = plain.build_draft_tree(parents, starts, np.array([3, 6]), table, 4, lambda p: max(0, p - 1), 1)
    assert got[1].tolist() == [2, 3, 3, 4]
    assert got[4].tolist() == [[0b1], [0b11], [0b101], [0b1100]]


def test_a_chain_sees_what_causal_attention_sees() -> None:
    b = tree_batch([5], [6], q_heads=2, kv_heads=1, dim=4, block_size=4, shape="chain", dtype=torch.float32)
    meta = plain.build_draft_tree(b.parents.numpy(), b.starts.numpy(), b.committed.numpy(), b.table.numpy(), 4, full, 1)
    out, _, _ = plain.tree_attention(b.query.numpy(), b.cache.numpy(), meta[1], b.starts.numpy(), meta[2],
                                     b.table.numpy(), meta[4], 0.5)
    keys, values = (b.cache[i][b.table[0]].reshape(-1, 4)[:11].double() for i in range(2))
    score = torch.einsum("nhd,kd->nhk", b.query.double(), keys) * 0.5
    score.masked_fill_(torch.arange(11)[None, None] > 6 + torch.arange(5)[:, None, None], -torch.inf)
    expected = torch.softmax(score, 2) @ values
    np.testing.assert_allclose(out, expected.numpy(), rtol=1e-12)


def test_acceptance_of_a_known_tree() -> None:
    parents, starts = np.array([-1, 0, 0, 2, 2, 0, 5]), np.array([0, 7])
    draft = np.array([9, 4, 6, 1, 2, 6, 2])
    target = np.array([6, 0, 2, 0, 8, 2, 3])
    # 0 -> target 6: nodes 2 and 5, the first; 2 -> target 2: node 4; it ends.
    nodes, count, tokens, lengths, last = plain.accept_draft_tree(draft, target, parents, starts, np.array([10]), 5)
    assert nodes.tolist() == [[0, 2, 4, -1, -1]] and count.tolist() == [3]
    assert tokens.tolist() == [[6, 2, 8, -1, -1]] and lengths.tolist() == [13] and last.tolist() == [4]
    nodes, count, *_ = plain.accept_draft_tree(draft, target, parents, starts, np.array([10]), 2)
    assert nodes.tolist() == [[0, 2]] and count.tolist() == [2]


def test_moved_rows_of_a_known_path() -> None:
    cache = np.arange(2 * 3 * 4, dtype=np.float64).reshape(2, 3, 4, 1, 1)
    moved = plain.compact_draft_kv(cache, np.array([[2, 0]]), np.array([2]), np.array([[0, 2, 3, -1]]), np.array([3]))
    assert moved[0, :, :, 0, 0].tolist() == [[1, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 0]]
    assert moved[1, 2, :, 0, 0].tolist() == [20, 21, 22, 12]


def test_c_entries_refuse_before_touching_the_device(lib) -> None:
    ok, bad, shape, dtype = (_lib.MVB_OK, _lib.MVB_ERR_INVALID_ARGUMENT, _lib.MVB_ERR_UNSUPPORTED_SHAPE,
                             _lib.MVB_ERR_UNSUPPORTED_DTYPE)

    def tree(rows=4, requests=1, bs=16, kind=0, param=0, words=1, pointer=FAKE):
        return lib.mvb_build_draft_tree(pointer, FAKE, FAKE, FAKE, 8, 8, rows, requests, bs, kind, param, words,
                                        FAKE, FAKE, FAKE, FAKE, FAKE, None, None)

    assert tree(rows=-1) == tree(requests=-1) == tree(bs=0) == bad
    assert tree(words=0) == tree(words=17) == tree(kind=7) == tree(kind=1, param=0) == tree(pointer=None) == bad
    assert tree(rows=0, requests=0) == ok

    def attend(rows=4, requests=1, hq=4, hkv=2, d=128, words=1, dt=0, q=FAKE, scale=1.0):
        return lib.mvb_tree_attention(q, 512, 128, FAKE, FAKE, 4, 16, hkv, d, FAKE, FAKE, FAKE, FAKE, 8, 8, FAKE,
                                      words, rows, requests, hq, scale, dt, None, 0, None, None)

    assert attend(scale=0.0) == attend(scale=-1.0) == attend(scale=float("nan")) == attend(scale=float("inf")) == bad

    assert attend(dt=5) == dtype and attend(hq=3) == shape and attend(rows=0) == ok
    assert attend(rows=-1) == attend(requests=-1) == attend(words=0) == attend(words=17) == attend(q=None) == bad
    assert attend(hkv=0) == attend(d=0) == bad and attend(d=264, dt=2) == shape
    assert lib.mvb_tree_attention_workspace_size(-1, 1, 4, 2, 128) == 0
    assert lib.mvb_tree_attention_workspace_size(64, 4, 16, 8, 128) > 0

    def accept(rows=4, requests=1, most=4, p=FAKE):
        return lib.mvb_accept_draft_tree(p, FAKE, FAKE, FAKE, FAKE, rows, requests, most, FAKE, FAKE, FAKE, FAKE,
                                         FAKE, None, None)

    assert accept(rows=-1) == accept(requests=-1) == accept(most=0) == accept(most=1025) == accept(p=None) == bad
    assert accept(requests=0) == ok

    layers = (ctypes.c_void_p * 2)(256, 512)

    def move(n=2, nb=4, bs=16, hkv=2, d=8, dt=0, requests=1, most=4, caches=layers, nodes=FAKE):
        return lib.mvb_compact_draft_kv(caches, n, nb, bs, hkv, d, dt, FAKE, 8, 8, FAKE, nodes, FAKE, requests, most,
                                        None, None)

    assert move(dt=9) == dtype and move(n=0) == move(requests=0) == ok
    assert move(n=-1) == move(bs=0) == move(hkv=0) == move(d=0) == move(most=0) == move(most=1025) == bad
    assert move(caches=None) == move(nodes=None) == bad
    assert move(caches=(ctypes.c_void_p * 2)(256, 256)) == bad
    assert move(caches=(ctypes.c_void_p * 2)(256, None)) == move(caches=(ctypes.c_void_p * 2)(256, 257)) == bad


def test_the_capture_mode_is_one_of_three(lib) -> None:
    for mode in (-1, 3, 1 << 30):
        assert lib.mvb_exchange_capture_mode(ctypes.byref(ctypes.c_int32(mode))) == _lib.MVB_ERR_INVALID_ARGUMENT
    assert lib.mvb_exchange_capture_mode(None) == _lib.MVB_ERR_INVALID_ARGUMENT


def test_the_path_query_takes_any_arguments(lib) -> None:
    def path(bs=16, hkv=2, d=128, rows=4, requests=1, hq=4, dt=0, blocks=4, q=FAKE):
        return lib.mvb_tree_attention_uses_tcgen05(q, 512, 128, FAKE, FAKE, blocks, bs, hkv, d, rows, requests, hq, dt)

    assert path(bs=0) == path(hkv=0) == path(hq=0) == path(hq=3) == path(d=0) == path(rows=0) == path(rows=-1) == 0
    assert path(requests=-1) == path(blocks=0) == path(dt=2) == path(dt=7) == path(bs=48) == path(hq=130) == 0
    assert path(q=ctypes.c_void_p(264)) == path(blocks=1 << 30) == 0


def test_the_kv_move_refuses_caches_that_overlap(lib) -> None:
    """2 x 4 x 16 x 2 x 8 fp16 values are 4096 bytes."""

    def move(*at):
        caches = (ctypes.c_void_p * len(at))(*at)
        return lib.mvb_compact_draft_kv(caches, len(at), 4, 16, 2, 8, 0, FAKE, 8, 8, FAKE, FAKE, FAKE, 0, 4, None, None), \
            lib.mvb_compact_draft_kv(caches, len(at), 4, 16, 2, 8, 0, FAKE, 8, 8, FAKE, FAKE, FAKE, 1, 4, None, None)

    assert move(4096, 4096 + 4094) == move(8192, 256, 4608) == (_lib.MVB_OK, _lib.MVB_ERR_INVALID_ARGUMENT)


def test_entry_points_refuse_cpu_tensors() -> None:
    b = tree_batch([3, 2], [4, 5])
    with pytest.raises(RuntimeError, match="require CUDA tensors"):
        build_draft_tree(b.parents, b.starts, b.committed, b.table, 16)
    with pytest.raises(RuntimeError, match="require CUDA tensors"):
        accept_draft_tree(b.parents, b.parents, b.parents, b.starts, b.committed, max_accepted=2)
    with pytest.raises(RuntimeError, match="require CUDA tensors"):
        DraftKVCompactor([b.cache])
    with pytest.raises(ValueError, match="at least one"):
        DraftKVCompactor([])
    zero = torch.zeros(5, dtype=torch.int64)
    tree = DraftTree(AttentionMetadata(zero, zero, b.starts, b.committed, b.table, zero, 16), zero[:, None])
    operator = B200PagedAttentionOperator()
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        operator.attend_tree(b.query, b.cache, tree)
    with pytest.raises(RuntimeError, match="requires CUDA tensors"):
        operator.forward_tree(b.query, b.query, b.query, b.cache, tree)
