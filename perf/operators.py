"""Measured cases of the draft-tree operators: one speculative-decoding step.

A step verifies, for each of R requests, a tree of drafted tokens over the
request's paged KV cache: the tree's metadata is built on the device
(``build``), every node attends to the committed cache and its own ancestors
(``attend``), the target model's tokens pick the path that is kept
(``accept``), and the kept nodes' K/V rows move behind the committed ones in
every layer's cache (``compact``).

``run`` computes each operator in plain torch operations, or (``own`` true)
calls the framework.  Request r's sizes follow from the case alone; parents,
tokens, pages and values from the seed.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 16  # tokens of a KV page, as in the benchmark's configurations
GOLDEN, PLASTIC = 0.6180339887498949, 0.7548776662466927
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed() -> list[dict]:
    attend = {"op": "attend", "dim": 128, "window": 0}
    return [
        # Metadata of one user's small tree: pure launch latency.
        {"name": "build 1x8", "op": "build", "requests": 1, "nodes": 8, "ragged": False,
         "low": 257, "high": 257, "window": 0},
        # A full serving batch of ragged trees over a sliding-window layer group.
        {"name": "build 256x64 window", "op": "build", "requests": 256, "nodes": 64, "ragged": True,
         "low": 1, "high": 8192, "window": 1024},
        # One user's chat turn, a small tree over a short cache: latency.
        {"name": "attend 1x8 bf16", **attend, "requests": 1, "nodes": 8, "ragged": False,
         "low": 257, "high": 257, "q_heads": 16, "kv_heads": 8, "dtype": "bf16"},
        # A moderate batch of the 0.6B model's heads.
        {"name": "attend 32x16 fp16", **attend, "requests": 32, "nodes": 16, "ragged": False,
         "low": 512, "high": 4096, "q_heads": 16, "kv_heads": 8, "dtype": "fp16"},
        # A full batch, ragged trees (some requests draft nothing), 8B heads.
        {"name": "attend 64x32 bf16 ragged", **attend, "requests": 64, "nodes": 32, "ragged": True,
         "low": 1, "high": 8192, "q_heads": 32, "kv_heads": 8, "dtype": "bf16"},
        # Few long documents, wide trees: the split over the key axis.
        {"name": "attend 3x61 bf16 long", **attend, "requests": 3, "nodes": 61, "ragged": False,
         "low": 30000, "high": 65536, "q_heads": 32, "kv_heads": 8, "dtype": "bf16"},
        # The widest trees over a full batch: as much computing as reading.
        {"name": "attend 64x64 fp16 wide", **attend, "requests": 64, "nodes": 64, "ragged": False,
         "low": 4096, "high": 8192, "q_heads": 32, "kv_heads": 8, "dtype": "fp16"},
        # The exact path of an fp32 engine.
        {"name": "attend 5x24 fp32", **attend, "requests": 5, "nodes": 24, "ragged": True,
         "low": 100, "high": 1500, "q_heads": 16, "kv_heads": 8, "dtype": "fp32"},
        # The walk for a handful of users, and for a full batch of wide trees.
        {"name": "accept 4x16", "op": "accept", "requests": 4, "nodes": 16, "ragged": False, "keep": 8},
        {"name": "accept 512x64", "op": "accept", "requests": 512, "nodes": 64, "ragged": True, "keep": 16},
        # Every layer of the 0.6B model for one user, and for a full batch.
        {"name": "compact 1 user", "op": "compact", "requests": 1, "nodes": 24, "ragged": False, "low": 700,
         "high": 700, "layers": 28, "kv_heads": 8, "dim": 128, "dtype": "bf16", "keep": 8},
        {"name": "compact 256 users", "op": "compact", "requests": 256, "nodes": 32, "ragged": True, "low": 1,
         "high": 8192, "layers": 28, "kv_heads": 8, "dim": 128, "dtype": "fp16", "keep": 8},
    ]


def draw(rng) -> dict:
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    most: dict[str, float] = {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0.0), _cost(c))
    while True:
        op = rng.choice(("build", "attend", "attend", "attend", "accept", "compact"))
        case = {"op": op, "requests": spread(1, 512), "nodes": spread(1, 128), "ragged": rng.random() < 0.6}
        if op != "accept":
            case["high"] = spread(1, 65536)
            case["low"] = rng.randint(0, case["high"])
        if op in ("build", "attend"):
            case["window"] = rng.choice((0, 0, spread(1, 4096)))
        if op == "attend":
            case["kv_heads"] = rng.choice((1, 2, 3, 4, 8))
            case["q_heads"] = case["kv_heads"] * rng.choice((1, 2, 3, 4, 5, 8))
            case["dim"] = 128
            case["dtype"] = rng.choice(("bf16", "fp16", "bf16", "fp16", "fp32"))
        if op == "compact":
            case["layers"] = rng.randint(1, 40)
            case["kv_heads"] = rng.choice((1, 2, 3, 4, 8))
            case["dim"] = rng.choice((64, 96, 128))
            case["dtype"] = rng.choice(("bf16", "fp16", "fp32"))
        if op in ("accept", "compact"):
            case["keep"] = rng.randint(1, 16)
        if _cost(case) <= most[op] and sum(_lengths(case)[0]) > 0:
            return case


# ------------------------------------------------------------------ sizes
def _lengths(case) -> tuple[list[int], list[int]]:
    """(drafted nodes, committed tokens) of each request, spread evenly over
    the case's ranges; ragged trees go down to no node at all."""

    n, high, low = case["nodes"], case.get("high", 0), case.get("low", 0)
    nodes = [int((n + 1) * (((r + 1) * GOLDEN) % 1.0)) if case["ragged"] else n for r in range(case["requests"])]
    committed = [low + int((high - low + 1) * (((r + 1) * PLASTIC) % 1.0)) for r in range(case["requests"])]
    return nodes, committed


def _path(n: int) -> float:
    """Mean number of ancestors (itself among them) of a node of the random
    recursive tree of n nodes that ``prepare`` draws."""

    return 1.0 + max(0.0, math.log(n)) if n else 0.0


def work(case) -> dict:
    nodes, committed = _lengths(case)
    t, r, words = sum(nodes), case["requests"], -(-case["nodes"] // 64)
    if case["op"] == "build":
        # parents and table cells in; positions, starts, slots and masks out.
        return {"bytes": 8 * (t * (5 + words) + 3 * r), "flops": t}
    if case["op"] == "accept":
        return {"bytes": 8 * (3 * t + r * (2 * case["keep"] + 5)), "flops": t}
    if case["op"] == "compact":
        size = 4 if case["dtype"] == "fp32" else 2
        moved = sum(max(0.0, min(case["keep"], _path(n)) - 1.0) for n in nodes)  # the root stays in place
        rows = 2 * case["layers"] * moved
        return {"bytes": int(2 * rows * case["kv_heads"] * case["dim"] * size) + 8 * r * (case["keep"] + 3), "flops": 0}
    size = 4 if case["dtype"] == "fp32" else 2
    window = case["window"]
    # A request's queries together read one window and the tree; each reads its own.
    seen = [min(c, window - 1) if window else c for c in committed]
    keys = sum(c + n for c, n in zip(seen, nodes) if n)
    pairs = sum(n * (c + _path(n)) for c, n in zip(seen, nodes))
    d, hq, hkv = case["dim"], case["q_heads"], case["kv_heads"]
    return {"bytes": 2 * keys * hkv * d * size + 2 * t * hq * d * size + 8 * t * (1 + words) + 8 * keys // BLOCK,
            "flops": int(4 * d * hq * pairs)}


def _cost(case) -> float:
    """What a case costs, by what it moves and by what its plain form pads to."""

    w = work(case)
    nodes, committed = _lengths(case)
    cells = case["requests"] * case["nodes"] ** 2
    if case["op"] == "attend":
        cells = case["requests"] * (max(committed) + case["nodes"]) * (
            case["nodes"] * case["q_heads"] + case["kv_heads"] * case["dim"]) / 8
    if case["op"] == "compact":
        pages = sum(n // BLOCK + 2 for n in nodes)
        cells = case["layers"] * pages * BLOCK * case["kv_heads"] * case["dim"]
    return w["bytes"] + w["flops"] / 200 + cells


# ----------------------------------------------------------------- inputs
def prepare(case, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 2 + 1)
    nodes, committed = _lengths(case)
    n = torch.tensor(nodes, dtype=torch.int64, device=dev)
    c = torch.tensor(committed, dtype=torch.int64, device=dev)
    qsl = torch.zeros(len(nodes) + 1, dtype=torch.int64, device=dev)
    qsl[1:] = n.cumsum(0)
    request = torch.repeat_interleave(torch.arange(len(nodes), device=dev), n)
    local = torch.arange(request.numel(), device=dev) - qsl[request]
    t = request.numel()
    # A random recursive tree: each node's parent is any node before it.
    parents = (torch.rand(t, device=dev, generator=gen, dtype=torch.float64) * local).long().clamp(max=(local - 1).clamp(min=0))
    parents = torch.where(local == 0, -1, parents)
    state = {"case": dict(case), "op": case["op"], "qsl": qsl, "committed": c, "parents": parents}
    if case["op"] == "accept":
        # The target's token at every node, from a small vocabulary; a draft
        # token agrees with its parent's target token in about 6 of 10 nodes.
        target = torch.randint(0, 1000, (t,), device=dev, generator=gen)
        other = torch.randint(0, 1000, (t,), device=dev, generator=gen)
        agree = torch.rand(t, device=dev, generator=gen) < 0.6
        up = (qsl[request] + parents).clamp(min=0)
        state |= {"target": target, "draft": torch.where(agree & (local > 0), target[up], other)}
        return state
    if case["op"] == "compact":
        _prepare_compact(state, case, nodes, committed, gen)
        return state
    pages = -(-(c + n) // BLOCK)
    _table(state, pages, int(pages.sum()) + 3, gen)
    if case["op"] == "attend":
        dt = DTYPES[case["dtype"]]
        blocks = state["num_blocks"]
        state["cache"] = torch.empty((2, blocks, BLOCK, case["kv_heads"], case["dim"]), dtype=dt, device=dev)
        state["cache"].normal_(generator=gen)
        state["query"] = torch.empty((t, case["q_heads"], case["dim"]), dtype=dt, device=dev).normal_(generator=gen)
        state |= _plain_build(state)
    return state


def _table(state, pages, blocks: int, gen) -> None:
    """Each request's pages, drawn without replacement from the whole pool."""

    dev = pages.device
    width = max(1, int(pages.max()))
    chosen = torch.randperm(blocks, device=dev, generator=gen)[: int(pages.sum())]
    held = torch.arange(width, device=dev) < pages[:, None]
    table = torch.zeros((pages.numel(), width), dtype=torch.int64, device=dev)
    table[held] = chosen
    state |= {"table": table, "num_blocks": blocks}


def _prepare_compact(state, case, nodes, committed, gen) -> None:
    """Caches of every layer.  The pool holds each request's drafted pages;
    the committed pages before them are one shared prefix page (they are not
    touched)."""

    n, c, dev = state["qsl"].diff(), state["committed"], gen.device
    first, last = c // BLOCK, -(-(c + n) // BLOCK)
    held = torch.where(n > 0, last - first, 0)
    blocks = int(held.sum()) + 1
    width = max(1, int(last.max()))
    at = torch.arange(width, device=dev)
    table = torch.full((len(nodes), width), blocks - 1, dtype=torch.int64, device=dev)
    table[(at >= first[:, None]) & (at < last[:, None]) & (n > 0)[:, None]] = torch.randperm(blocks - 1, device=dev, generator=gen)
    caches = torch.empty((case["layers"], 2, blocks, BLOCK, case["kv_heads"], case["dim"]),
                         dtype=DTYPES[case["dtype"]], device=dev).normal_(generator=gen)
    # A kept path: the root, then increasing nodes, about as many as a random
    # recursive tree is deep.
    keep = case["keep"]
    step = torch.rand((len(nodes), keep), device=dev, generator=gen)
    path = torch.zeros((len(nodes), keep), dtype=torch.int64, device=dev)
    path[:, 1:] = (1 + (step[:, 1:] * n[:, None] / max(1.0, _path(case["nodes"]))).long()).cumsum(1)
    inside = path < n[:, None]
    state |= {"table": table, "caches": caches, "layers": list(caches.unbind(0)), "kept": inside.sum(1),
              "path": torch.where(inside, path, -1)}


# ------------------------------------------------------------ plain forms
def _dense(state):
    """Row of each [request, node] cell (clamped) and which cells are real."""

    qsl, width = state["qsl"], state["case"]["nodes"]
    at = torch.arange(width, device=qsl.device)
    real = at < qsl.diff()[:, None]
    return torch.where(real, qsl[:-1, None] + at, 0), real


def _closure(paths: torch.Tensor, steps: int) -> torch.Tensor:
    """Ancestor relation from the parent relation (with the identity), by
    squaring ``steps`` times."""

    return paths if steps == 0 else _closure((paths @ paths > 0).float(), steps - 1)


def _ancestors(state):
    """[R, N, N]: cell (i, j) says that node j is node i or an ancestor."""

    rows, real = _dense(state)
    parent = torch.where(real, state["parents"][rows], -1) if rows.numel() else rows
    at = torch.arange(real.shape[1], device=real.device)
    up = (parent[:, :, None] == at) & real[:, :, None]
    own_cell = (at[:, None] == at) & real[:, :, None]
    return _closure((up | own_cell).float(), max(1, real.shape[1] - 1).bit_length()) > 0, parent, real, rows


def _plain_build(state) -> dict:
    window = state["case"]["window"]
    anc, _, real, rows = _ancestors(state)
    c, table = state["committed"], state["table"]
    at = torch.arange(real.shape[1], device=c.device)
    position = c[:, None] + anc.sum(2) - 1
    start = (position - window + 1).clamp(min=0) if window else torch.zeros_like(position)
    logical = c[:, None] + at
    page = table.gather(1, (logical // BLOCK).clamp(max=table.shape[1] - 1))
    seen = anc & (position[:, None, :] >= start[:, :, None])
    words = -(-real.shape[1] // 64)
    bits = torch.zeros((*real.shape, words * 64), dtype=torch.int64, device=c.device)
    bits[:, :, : real.shape[1]] = seen.long()
    weight = torch.ones(64, dtype=torch.int64, device=c.device) << torch.arange(64, device=c.device)
    mask = (bits.view(*real.shape, words, 64) * weight).sum(3)
    return {"positions": position[real], "starts": start[real], "lengths": c + state["qsl"].diff(),
            "slots": (page * BLOCK + logical % BLOCK)[real], "mask": mask[real]}


def _plain_attend(state) -> torch.Tensor:
    case, cache, c = state["case"], state["cache"], state["committed"]
    rows, real = _dense(state)
    hkv, dim = case["kv_heads"], case["dim"]
    group = case["q_heads"] // hkv
    r, n = real.shape
    keys, values = cache[0][state["table"]], cache[1][state["table"]]
    size = keys.shape[1] * BLOCK
    q = state["query"][rows].view(r, n, hkv, group, dim).permute(0, 2, 1, 3, 4).float()
    k = keys.view(r, size, hkv, dim).permute(0, 2, 3, 1).float()
    score = (q.reshape(r, hkv, n * group, dim) @ k) / math.sqrt(dim)
    at = torch.arange(size, device=c.device)
    node = at - c[:, None]
    inside = (node >= 0) & (node < state["qsl"].diff()[:, None])
    node = torch.where(inside, node, 0)
    words = state["mask"][rows]
    picked = words.gather(2, (node // 64)[:, None, :].expand(r, n, size))
    drafted = ((picked >> (node % 64)[:, None, :]) & 1 > 0) & inside[:, None, :]
    start = torch.maximum(state["starts"][rows], state["starts"][rows[:, :1]])
    committed = (at < c[:, None, None]) & (at >= start[:, :, None])
    seen = ((committed | drafted) & real[:, :, None])[:, None, :, None, :].expand(r, hkv, n, group, size)
    score = score.masked_fill(~seen.reshape(score.shape), -torch.inf)
    top = score.amax(3, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = torch.exp(score - top)
    total = weight.sum(3, keepdim=True)
    v = values.view(r, size, hkv, dim).permute(0, 2, 1, 3).float()
    out = (weight @ v) / torch.where(total > 0, total, 1.0)
    return out.view(r, hkv, n, group, dim).permute(0, 2, 1, 3, 4)[real].reshape(-1, hkv * group, dim).to(cache.dtype)


def _plain_accept(state):
    keep, draft, target = state["case"]["keep"], state["draft"], state["target"]
    anc, parent, real, rows = _ancestors(state)
    n = real.shape[1]
    tok, want = draft[rows], target[rows]
    at = torch.arange(n, device=rows.device)
    same = (parent[:, :, None] == parent[:, None, :]) & (tok[:, :, None] == tok[:, None, :])
    twin = (same & (at[None, :] < at[:, None]) & real[:, None, :]).any(2)
    agrees = (tok == want.gather(1, parent.clamp(min=0))) & (parent >= 0) & ~twin
    agrees = (agrees | (at == 0)) & real
    depth = anc.sum(2) - 1
    kept = real & ~(anc & ~agrees[:, None, :]).any(2) & (depth < keep)
    count = kept.sum(1)
    place = torch.where(kept, depth, keep)
    path = torch.full((real.shape[0], keep + 1), -1, dtype=torch.int64, device=rows.device)
    path.scatter_(1, place, at.expand_as(place))
    out = torch.full_like(path, -1).scatter_(1, place, want)
    path, out = path[:, :keep], out[:, :keep]
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])[:, 0]
    return {"nodes": path, "count": count, "tokens": out, "lengths": state["committed"] + count,
            "rows": torch.where(count > 0, state["qsl"][:-1] + last, -1)}


def _plain_compact(state) -> torch.Tensor:
    path, c, table, caches = state["path"], state["committed"], state["table"], state["caches"]
    at = torch.arange(path.shape[1], device=path.device)
    moves = (path >= 0) & (path != at)
    source, goal = (c[:, None] + path).clamp(min=0), c[:, None] + at
    cells = lambda p: (table.gather(1, (p // BLOCK).clamp(max=table.shape[1] - 1)) * BLOCK + p % BLOCK)[moves]  # noqa: E731
    rows = caches.view(caches.shape[0], 2, -1, *caches.shape[4:])
    rows[:, :, cells(goal)] = rows[:, :, cells(source)]
    return _bits(caches)


def _bits(caches: torch.Tensor) -> torch.Tensor:
    """A move keeps every bit: the caches as whole numbers."""

    return caches.view(torch.int32 if caches.dtype == torch.float32 else torch.int16)


# -------------------------------------------------------------------- run
_kept: dict = {}


def _framework():
    """The framework's entry points, and the operator that a program keeps."""

    if not _kept:
        import micro_vllm_b200 as framework

        _kept["framework"] = framework
        _kept["operator"] = framework.B200PagedAttentionOperator()
        _kept["full"] = framework.FullAttentionSpec()
    return _kept["framework"]


def run(state):
    op = state["op"]
    if not own:
        if op == "build":
            return _plain_build(state)
        if op == "attend":
            return _plain_attend(state)
        return _plain_accept(state) if op == "accept" else _plain_compact(state)
    framework = _framework()
    case = state["case"]
    if op == "build":
        spec = framework.SlidingWindowSpec(case["window"]) if case["window"] else _kept["full"]
        tree = framework.build_draft_tree(state["parents"], state["qsl"], state["committed"], state["table"],
                                          BLOCK, spec=spec, max_nodes=case["nodes"])
        md = tree.attention
        return {"positions": md.query_positions, "starts": md.query_context_start_positions,
                "lengths": md.context_lengths, "slots": md.slot_mapping, "mask": tree.ancestor_mask}
    if op == "attend":
        metadata = framework.AttentionMetadata(
            query_positions=state["positions"], query_context_start_positions=state["starts"],
            query_start_locations=state["qsl"], context_lengths=state["lengths"], block_table=state["table"],
            slot_mapping=state["slots"], block_size=BLOCK)
        tree = framework.DraftTree(attention=metadata, ancestor_mask=state["mask"])
        return _kept["operator"].attend_tree(state["query"], state["cache"], tree)
    if op == "accept":
        kept = framework.accept_draft_tree(state["draft"], state["target"], state["parents"], state["qsl"],
                                           state["committed"], max_accepted=case["keep"])
        return {"nodes": kept.nodes, "count": kept.num_accepted, "tokens": kept.tokens,
                "lengths": kept.committed_lengths, "rows": kept.last_rows}
    if "mover" not in state:  # made once for the caches of a program's layers
        state["mover"] = framework.DraftKVCompactor(state["layers"])
    state["mover"](state["table"], state["committed"], state["path"], state["kept"])
    return _bits(state["caches"])


# ------------------------------------------------------------------ exact
def exact(case, seed: int):
    """Attention in 64 bits, one request at a time over its own keys only;
    the other operators give whole numbers, which have to be equal."""

    if case["op"] != "attend":
        return None
    nodes, committed = _lengths(case)
    if sum(n * (c + n) for n, c in zip(nodes, committed)) * case["q_heads"] * case["dim"] > 1 << 41:
        return None
    state = prepare(case, seed)
    qsl = state["qsl"].tolist()
    words, parents, starts = state["mask"].tolist(), state["parents"].tolist(), state["starts"].tolist()
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device=state["query"].device)
    for r, (n, c) in enumerate(zip(nodes, committed)):
        if n == 0:
            continue
        first = qsl[r]
        at = torch.arange(c + n, device=out.device)
        block = state["table"][r, at // BLOCK]
        key, value = (plane[block, at % BLOCK].double() for plane in state["cache"])  # [S, Hkv, D]
        seen = torch.zeros((n, c + n), dtype=torch.bool)
        for i in range(n):
            seen[i, starts[first + i]: c] = True
            depth, j = words[first + i], i
            while j >= 0:  # walk to the root; the window may end the walk early
                seen[i, c + j] = bool((depth[j // 64] >> (j % 64)) & 1)
                j = parents[first + j]
        seen = seen.to(out.device)
        group = case["q_heads"] // case["kv_heads"]
        for h in range(case["kv_heads"]):
            q = state["query"][first: first + n, h * group: (h + 1) * group].double()
            s = torch.einsum("ngd,sd->ngs", q, key[:, h]) * case["dim"] ** -0.5
            p = torch.where(seen[:, None, :], (s - s.max()).exp(), 0.0)
            p /= p.sum(2, keepdim=True)
            out[first: first + n, h * group: (h + 1) * group] = torch.einsum("ngs,sd->ngd", p, value[:, h])
    return out
