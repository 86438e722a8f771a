"""Workloads of drafted trees over the pages of a ledger, and of rotary positions.

A step of drafting: a model proposes a tree of rows behind each sequence of a paged KV history, one
pass verifies all of them at once, and the rows of one accepted path become history. The operators
are those of that step: the tree's ancestor bits and positions, the append of the rows' keys and
values to the pages with the rotation of keys and queries on the way, the attention of every drafted
row to the history and its own ancestors, the move of the accepted rows; and the rotation of any
tensor of heads by itself.

``run`` computes a pass either in plain torch operations in 32 bits (angles in 64) or, where ``own``
is true, through the framework's entry points in ``h3sa.drafts`` and ``h3sa.rotary``. ``exact`` is
the definition in 64 bits, written apart from both.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

PAGE = 128  # rows of a page
DIM = 128  # head dimension of the caches
ROOT = Path(__file__).resolve().parents[1]


def listed() -> list[dict]:
    return [
        # A handful of drafts behind two short streams, three local heads (an eighth of 24): the
        # smallest verification, where launches and latency are everything.
        dict(name="attend_two_streams", op="attend", batch=2, nodes=9, heads=3, kv_heads=3, shared=0,
             history=311, kind="bf16", lse=False),
        # Twenty candidate continuations of one document with a small tree each, idle slots among them.
        dict(name="attend_shared_document", op="attend", batch=20, nodes=13, heads=32, kv_heads=8, shared=8192,
             history=700, kind="bf16", lse=True),
        # Trees behind histories that nobody shares: bound by reading each history once.
        dict(name="attend_own_histories", op="attend", batch=24, nodes=24, heads=32, kv_heads=8, shared=0,
             history=9000, kind="bf16", lse=False),
        # Wide trees over long e4m3 histories, five query heads a KV head: bound by arithmetic.
        dict(name="attend_e4m3_wide_trees", op="attend", batch=4, nodes=127, heads=40, kv_heads=8, shared=0,
             history=24001, kind="e4m3", lse=False),
        # One new token behind each of two streams: the smallest append.
        dict(name="append_two_tokens", op="append", batch=2, rows=1, heads=3, kv_heads=3, history=311,
             rotary=128, interleaved=False, base=10000.0, far=0, kind="bf16"),
        # Prompt chunks of several requests, ragged, into an e4m3 cache; half of each head rotated, in
        # pairs, at far positions: bound by memory.
        dict(name="append_e4m3_prompts", op="append", batch=7, rows=3001, heads=32, kv_heads=8, history=900,
             rotary=64, interleaved=True, base=1000000.0, far=250000, kind="e4m3"),
        # Queries of a small batch, an odd number of rows and heads of 64.
        dict(name="rotate_few_rows", op="rotate", tokens=57, heads=14, dim=64, rotary=64, axes=1,
             interleaved=True, base=10000.0, far=2000, kind="fp16"),
        # Queries of a whole video chunk on three position axes (time, height, width), 96 of 128
        # dimensions rotated: bound by memory.
        dict(name="rotate_video_chunk", op="rotate", tokens=24605, heads=24, dim=128, rotary=96, axes=3,
             interleaved=False, base=10000.0, far=4000, kind="bf16"),
        # The trees of two streams.
        dict(name="tree_two_streams", op="tree", batch=2, nodes=9),
        # Large trees for many requests at once.
        dict(name="tree_many_requests", op="tree", batch=64, nodes=500),
        # An accepted path of one layer.
        dict(name="keep_one_layer", op="keep", tensors=2, heads=3, batch=2, nodes=9, history=311),
        # Accepted paths of many requests in K and V of fifty layers.
        dict(name="keep_all_layers", op="keep", tensors=100, heads=3, batch=24, nodes=64, history=500),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["attend", "attend", "attend", "append", "append", "rotate", "rotate", "tree", "keep"])
    if op == "tree":
        return dict(op=op, batch=_log(rng, 1, 64), nodes=_log(rng, 1, 500))
    if op == "keep":
        layers = _log(rng, 1, 50)
        return dict(op=op, tensors=2 * layers, heads=rng.choice([1, 2, 3, 6, 8]) if layers < 15 else rng.choice([1, 2, 3]),
                    batch=_log(rng, 1, 24), nodes=_log(rng, 1, 64), history=_log(rng, 1, 500))
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    base = rng.choice([10000.0, 500000.0, 1000000.0])
    if op == "append":
        rows = _log(rng, 1, 3001) if rng.random() < 0.5 else _log(rng, 1, 40)
        heads = kv_heads * group
        batch = _log(rng, 1, max(1.0, min(64.0, 21000 * 48 / (rows * (heads + 2 * kv_heads)))))
        return dict(op=op, batch=batch, rows=rows, heads=heads if rng.random() < 0.8 else 0, kv_heads=kv_heads,
                    history=_log(rng, 1, 900), rotary=rng.choice([128, 128, 64, 96, 32, 0]),
                    interleaved=rng.random() < 0.5, base=base, far=rng.choice([0, 0, 9000, 250000]),
                    kind=rng.choice(["bf16", "bf16", "e4m3"]))
    if op == "rotate":
        axes = rng.choice([1, 1, 3])
        dim = rng.choice([64, 72, 80, 96, 128, 128, 192, 256])
        heads = _log(rng, 1, 40)
        rotary = rng.choice([r for r in (24, 48, 64, 72, 96, 120, 128, 192, 256) if r <= dim and r % (2 * axes) == 0])
        kind = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        most = 24605 * 24 * 128 * 2 / (heads * dim * (4 if kind == "fp32" else 2))
        return dict(op=op, tokens=_log(rng, 1, most), heads=heads, dim=dim, rotary=rotary, axes=axes,
                    interleaved=rng.random() < 0.5, base=base, far=rng.choice([0, 4000, 1000000]), kind=kind)
    while True:
        case = dict(op=op, batch=_log(rng, 1, 64), nodes=_log(rng, 1, 128), heads=kv_heads * group, kv_heads=kv_heads,
                    shared=PAGE * _log(rng, 1, 300) if rng.random() < 0.3 else 0, history=_log(rng, 1, 30000),
                    kind=rng.choice(["bf16", "bf16", "e4m3"]), lse=rng.random() < 0.3)
        keys = case["shared"] + case["history"] + case["nodes"]
        # no more arithmetic, and no more cache, than the largest listed calls
        scores = case["batch"] * case["nodes"] * case["heads"] * keys
        cells = kv_heads * case["batch"] * keys
        if scores <= 4.5e8 and cells <= 1.7e6:
            return case


# ------------------------------------------------------------------------------------ inputs


def _dev(a: np.ndarray, dtype: torch.dtype = torch.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def _normal(gen: torch.Generator, *shape: int, dtype: torch.dtype = torch.bfloat16, spread: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, device="cuda").normal_(0.0, spread, generator=gen).to(dtype)


def _trees(rs: np.random.RandomState, batch: int, nodes: int) -> tuple[np.ndarray, np.ndarray]:
    """Drafted trees as a drafting model leaves them: level by level, each level a few of the last
    level's continuations, one root (now and then several). parents [batch, nodes], -1 for a root;
    counts [batch]: nodes that a sequence has, the rest of its row is unused."""

    parents = np.full((batch, nodes), -1, np.int64)
    counts = rs.randint(max(1, nodes // 2), nodes + 1, batch)
    counts[rs.randint(batch)] = nodes
    for b in range(batch):
        lo, hi = 0, min(nodes, 1 if rs.rand() < 0.8 else 3)  # the last level
        while hi < nodes:
            width = min(nodes - hi, rs.randint(1, max(2, nodes // 6) + 1))
            parents[b, hi:hi + width] = np.sort(rs.randint(lo, hi, width))
            lo, hi = hi, hi + width
    return parents, counts


def _ancestors(parents: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """sees [batch, nodes, nodes]: whether a node is another or one of its ancestors; depths."""

    batch, nodes = parents.shape
    sees = np.zeros((batch, nodes, nodes), bool)
    at = np.arange(batch)
    for i in range(nodes):
        p = parents[:, i]
        sees[:, i] = np.where((p >= 0)[:, None], sees[at, np.maximum(p, 0)], False)
        sees[:, i, i] = True
    return sees, sees.sum(-1) - 1


def _words(sees: np.ndarray) -> np.ndarray:
    """Truth values [..., n] as 32-bit words [..., ceil(n / 32)], the lowest bit first."""

    wide = np.zeros((*sees.shape[:-1], -(-sees.shape[-1] // 32) * 32), np.uint8)
    wide[..., :sees.shape[-1]] = sees
    return np.packbits(wide, axis=-1, bitorder="little").view("<u4").astype(np.uint32).view(np.int32)


def _pages(rs: np.random.RandomState, rows: np.ndarray, shared: int = 0, most: int = 0) -> tuple[np.ndarray, int]:
    """Table of sequences with pages for `rows` rows, scattered over the pool; the first `shared`
    pages are the same for all that have any. Returns it and the pool's pages, which are as many as
    sequences of `most` rows would need where that is given."""

    held = -(-rows // PAGE)
    mine = np.where(held > 0, np.maximum(held - shared, 0), 0)
    pages = (len(rows) * -(-most // PAGE) if most else shared + int(mine.sum())) + 3
    ids = rs.permutation(pages)
    table = np.full((len(rows), max(1, int(held.max()))), -1, np.int64)
    at = shared
    for b, n in enumerate(held):
        if n:
            table[b, :shared] = ids[:shared]
            table[b, shared:n] = ids[at:at + mine[b]]
            at += mine[b]
    return table, pages


def _e4m3_pools(gen: torch.Generator, state: dict, shape: tuple[int, ...]) -> None:
    for name in ("k", "v"):
        x = _normal(gen, *shape)
        scale = x.abs().amax(dim=(1, 2)).float() / 448.0
        state[name + "_scale"] = scale
        state[name] = (x.float() / scale[:, None, None]).to(torch.float8_e4m3fn)


def _frequencies(case: dict) -> torch.Tensor:
    """What a program makes once per model: radians a position of every pair, [axes, pairs of an axis]."""

    axes = case.get("axes", 1)
    pairs = case["rotary"] // 2 // axes
    one = case["base"] ** (-np.arange(pairs, dtype=np.float64) / max(1, pairs))
    return _dev(np.tile(one, (axes, 1)), torch.float64)


def prepare(case: dict, seed: int) -> dict:
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case=case)
    batch = case.get("batch", 1)
    if case["op"] == "rotate":
        kind = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)[case["kind"]]
        s["x"] = _normal(gen, case["tokens"], case["heads"], case["dim"], dtype=kind, spread=1.5)
        if case["axes"] == 1:  # rows of several sequences one after another
            at = case["far"] + np.arange(case["tokens"]) % max(1, case["tokens"] // 3)
            s["positions"] = _dev(at, torch.int32)
        else:  # frames of a grid; height and width in fractions of the frame
            frame = 17
            t = np.arange(case["tokens"])
            grid = np.stack([case["far"] + t // (frame * frame) * (20 / 3), t // frame % frame * (32 / frame), t % frame * (32 / frame)], -1)
            s["positions"] = _dev(grid[:, :case["axes"]], torch.float64)
        s["frequencies"] = _frequencies(case)
        return s
    if case["op"] == "append":
        counts = rs.randint(max(1, case["rows"] // 3), case["rows"] + 1, batch)
        counts[rs.randint(batch)] = case["rows"]
        lengths = rs.randint(0, case["history"] + 1, batch)
        table, pages = _pages(rs, lengths + counts, most=case["history"] + case["rows"])
        kv = (batch, case["rows"], case["kv_heads"], DIM)
        s["key"], s["value"] = _normal(gen, *kv, spread=1.5), _normal(gen, *kv)
        if case["heads"]:
            s["query"] = _normal(gen, batch, case["rows"], case["heads"], DIM, spread=1.5)
        shape = (case["kv_heads"], pages * PAGE, DIM)
        if case["kind"] == "e4m3":
            _e4m3_pools(gen, s, shape)
        else:
            s["k"], s["v"] = _normal(gen, *shape), _normal(gen, *shape)
        s["positions"] = _dev(case["far"] + lengths[:, None] + np.arange(case["rows"]))
        s["frequencies"] = _frequencies(case)
        s["counts"], s["lengths"], s["table"] = _dev(counts), _dev(lengths), _dev(table)
        return s
    parents, counts = _trees(rs, batch, case["nodes"])
    if case["op"] == "tree":
        s["parents"], s["counts"] = _dev(parents), _dev(counts)
        s["lengths"] = _dev(rs.randint(0, 30000, batch))
        return s
    if case["op"] == "keep":
        lengths = rs.randint(0, case["history"] + 1, batch)
        table, pages = _pages(rs, lengths + counts, most=case["history"] + case["nodes"])
        path = np.full((batch, case["nodes"]), -1, np.int64)
        for b in range(batch):
            # the accepted path: up to some drafted row; of the rows that would lie where another
            # comes to lie (a second pass over the same inputs would read them), none
            for leaf in rs.permutation(counts[b]):
                found = [int(leaf)]
                while parents[b, found[-1]] >= 0:
                    found.append(int(parents[b, found[-1]]))
                found = found[::-1]
                if all(n == k or n >= len(found) for k, n in enumerate(found)):
                    path[b, :len(found)] = found
                    break
        s["pools"] = _normal(gen, case["tensors"], case["heads"], pages * PAGE, DIM)
        s["path"], s["lengths"], s["table"] = _dev(path), _dev(lengths), _dev(table)
        return s
    lengths = case["shared"] + rs.randint(case["history"] // 4, case["history"] + 1, batch)
    lengths[rs.randint(batch)] = case["shared"] + case["history"]
    if batch > 4:
        idle = rs.randint(batch, size=batch // 5)  # slots without a sequence
        lengths[idle] = counts[idle] = 0
    table, pages = _pages(rs, lengths + counts, case["shared"] // PAGE)
    sees, _ = _ancestors(parents)
    sees &= (np.arange(case["nodes"]) < counts[:, None])[:, :, None]
    s["query"] = _normal(gen, batch, case["nodes"], case["heads"], DIM, spread=1.5)
    shape = (case["kv_heads"], pages * PAGE, DIM)
    if case["kind"] == "e4m3":
        _e4m3_pools(gen, s, shape)
    else:
        s["k"], s["v"] = _normal(gen, *shape), _normal(gen, *shape)
    s["masks"] = _dev(_words(sees))
    s["counts"], s["lengths"], s["table"] = _dev(counts), _dev(lengths), _dev(table)
    return s


# ------------------------------------------------------------------------------ plain forms


def _turned(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x [..., heads, dim] rotated at positions [...] or [..., axes], in 32 bits (angles in 64)."""

    pairs = frequencies.numel()
    if pairs == 0:
        return x.float()
    where = positions.double()
    angle = (where[..., None] * frequencies[0] if where.ndim < x.ndim - 1
             else (where[..., None] * frequencies).flatten(-2))
    cos, sin = torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]
    x = x.float()
    turned, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)
    a, b = turned[..., :pairs], turned[..., pairs:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)


def _rotate_plain(s: dict) -> torch.Tensor:
    return _turned(s["x"], s["positions"], s["frequencies"], s["case"]["interleaved"]).to(s["x"].dtype)


def _append_plain(s: dict) -> dict:
    c = s["case"]
    at = torch.arange(c["rows"], device="cuda")
    row = s["lengths"].long()[:, None] + at
    live = (at < s["counts"][:, None]).view(-1)
    page = s["table"].long().gather(1, (row // PAGE).clamp(max=s["table"].shape[1] - 1))
    dst = (page * PAGE + row % PAGE).view(-1)[live]
    key = _turned(s["key"], s["positions"], s["frequencies"], c["interleaved"])
    for name, new in (("k", key), ("v", s["value"].float())):
        new = new.view(-1, c["kv_heads"], DIM)[live].transpose(0, 1)
        if c["kind"] == "e4m3":
            new = (new / s[name + "_scale"][:, None, None]).clamp(-448.0, 448.0)
        raw = s[name].view(torch.uint8 if c["kind"] == "e4m3" else torch.int16)
        raw[:, dst] = new.to(s[name].dtype).view(raw.dtype)
    out = {"k": s["k"], "v": s["v"]}
    if c["heads"]:
        out["query"] = _turned(s["query"], s["positions"], s["frequencies"], c["interleaved"]).to(s["query"].dtype)
        out["query"] = torch.where(live.view(c["batch"], -1, 1, 1), out["query"], 0.0)
    return out


def _tree_plain(s: dict) -> dict:
    batch, nodes = s["parents"].shape
    at = torch.arange(nodes, device="cuda")
    reach = (at == s["parents"][:, :, None]) | (at == at[:, None])
    for _ in range(max(1, (nodes - 1).bit_length())):  # paths of twice the length
        reach = torch.matmul(reach.float(), reach.float()) > 0
    live = at < s["counts"][:, None]
    reach = reach & live[:, :, None]
    depth = reach.sum(-1) - 1
    positions = torch.where(live, s["lengths"][:, None] + depth, 0)
    words = -(-nodes // 32)
    bits = torch.zeros(batch, nodes, words * 32, dtype=torch.int64, device="cuda")
    bits[:, :, :nodes] = reach
    value = (bits.view(batch, nodes, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    value = torch.where(value >= 1 << 31, value - (1 << 32), value)
    return {"masks": value.int(), "positions": positions.int()}


def _keep_plain(s: dict) -> dict:
    c = s["case"]
    path, lengths = s["path"].long(), s["lengths"].long()
    kept = path >= 0
    step = torch.arange(path.shape[1], device="cuda")

    def place(row: torch.Tensor) -> torch.Tensor:
        page = s["table"].long().gather(1, (row // PAGE).clamp(0, s["table"].shape[1] - 1))
        return (page * PAGE + row % PAGE)[kept]

    src, dst = place(lengths[:, None] + path), place(lengths[:, None] + step)
    s["pools"][:, :, dst] = s["pools"][:, :, src]
    return {"pools": s["pools"], "lengths": (lengths + kept.sum(1)).int()}


def _attend_plain(s: dict) -> dict:
    c = s["case"]
    batch, nodes, heads, kv = c["batch"], c["nodes"], c["heads"], c["kv_heads"]
    group = heads // kv
    width = s["table"].shape[1]
    table, lengths, counts = s["table"].long(), s["lengths"].long(), s["counts"].long()

    def rows_of(name: str) -> torch.Tensor:  # [kv, batch, width * PAGE, dim]
        pool = s[name].view(torch.uint8).view(kv, -1, PAGE * DIM * s[name].element_size())
        x = pool[:, table.clamp(min=0)].view(s[name].dtype).view(kv, batch, width * PAGE, DIM).float()
        return x * s[name + "_scale"][:, None, None, None] if c["kind"] == "e4m3" else x

    k, v = rows_of("k"), rows_of("v")
    at = torch.arange(width * PAGE, device="cuda")
    v = torch.where((at < (lengths + counts)[:, None])[None, :, :, None], v, 0.0)
    node = at - lengths[:, None]  # which drafted row a key is
    word = s["masks"].long().gather(2, (node // 32).clamp(0, s["masks"].shape[2] - 1)[:, None].expand(-1, nodes, -1))
    drafted = (word >> (node % 32)[:, None] & 1) == 1
    seen = (node < 0)[:, None] | (drafted & (node < counts[:, None])[:, None])
    seen = seen & (torch.arange(nodes, device="cuda") < counts[:, None])[:, :, None]
    seen = seen.repeat_interleave(group, 1)  # [batch, nodes * group, keys]
    q = s["query"].float().view(batch, nodes, kv, group, DIM).permute(2, 0, 1, 3, 4).reshape(kv, batch, nodes * group, DIM)
    x = torch.where(seen, torch.matmul(q * DIM ** -0.5, k.transpose(2, 3)), float("-inf"))
    top = x.amax(-1, keepdim=True)
    base = torch.where(top.isinf(), 0.0, top)
    p = torch.exp(x - base)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, torch.matmul(p, v) / total, 0.0)
    back = lambda t: t.view(kv, batch, nodes, group, -1).permute(1, 2, 0, 3, 4).reshape(batch, nodes, heads, -1)  # noqa: E731
    out = {"out": back(o).bfloat16()}
    if c["lse"]:
        out["lse"] = back(base + torch.log(total)).squeeze(-1)
    return out


# ------------------------------------------------------------------------ the framework's own


def _module(name: str):
    at = str(ROOT / "taomate-h3_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import importlib

    return importlib.import_module("h3sa." + name)


def _own(s: dict) -> object:
    c = s["case"]
    if c["op"] == "rotate":
        return _module("rotary").rotate(s["x"], s["positions"], s["frequencies"], interleaved=c["interleaved"])
    ops = _module("drafts")
    if c["op"] == "append":
        query = ops.append_rows(s["key"], s["value"], s["k"], s["v"], s["table"], s["lengths"], counts=s["counts"],
                                positions=s["positions"], frequencies=s["frequencies"] if c["rotary"] else None,
                                interleaved=c["interleaved"], query=s.get("query"), k_scale=s.get("k_scale"),
                                v_scale=s.get("v_scale"))
        return {"k": s["k"], "v": s["v"]} if query is None else {"k": s["k"], "v": s["v"], "query": query}
    if c["op"] == "tree":
        masks, positions = ops.draft_tree(s["parents"], s["lengths"], counts=s["counts"])
        return {"masks": masks, "positions": positions}
    if c["op"] == "keep":
        return {"pools": s["pools"], "lengths": ops.keep_rows(s["pools"], s["table"], s["lengths"], s["path"])}
    lse = torch.empty(c["batch"], c["nodes"], c["heads"], device="cuda") if c["lse"] else None
    out = ops.tree_attention(s["query"], s["k"], s["v"], s["table"], s["lengths"], s["masks"], DIM ** -0.5,
                             counts=s["counts"], shared_rows=c["shared"], k_scale=s.get("k_scale"),
                             v_scale=s.get("v_scale"), lse=lse)
    return {"out": out} if lse is None else {"out": out, "lse": lse}


def run(state: dict) -> object:
    if own:
        return _own(state)
    plain = {"attend": _attend_plain, "append": _append_plain, "rotate": _rotate_plain, "tree": _tree_plain,
             "keep": _keep_plain}
    return plain[state["case"]["op"]](state)


# ---------------------------------------------------------------------------- cost and truth


def work(case: dict) -> dict:
    """Mean figures of the drawn inputs (their exact lengths depend on the seed)."""

    batch = case.get("batch", 1)
    if case["op"] == "rotate":
        values = case["tokens"] * case["heads"] * case["dim"]
        size = 4 if case["kind"] == "fp32" else 2
        return {"bytes": 2.0 * size * values + case["tokens"] * (4 if case["axes"] == 1 else 8 * case["axes"]),
                "flops": 3.0 * case["tokens"] * case["heads"] * case["rotary"]}
    if case["op"] == "append":
        rows = batch * (case["rows"] * 2 / 3)
        size = 1 if case["kind"] == "e4m3" else 2
        return {"bytes": DIM * (rows * (2 * case["kv_heads"] * (2 + size) + 2 * case["heads"])
                                + 2 * batch * case["rows"] * case["heads"]) + 4.0 * batch * case["rows"],
                "flops": 3.0 * rows * (case["kv_heads"] + case["heads"]) * case["rotary"]}
    nodes = case["nodes"]
    if case["op"] == "tree":
        return {"bytes": 4.0 * batch * nodes * (2 + -(-nodes // 32)), "flops": 0.0}
    if case["op"] == "keep":
        moved = batch * 0.09 * nodes ** 0.73  # of the paths that prepare() makes
        return {"bytes": 4.0 * case["tensors"] * case["heads"] * DIM * moved + 4.0 * batch * (2 + nodes), "flops": 0.0}
    live = 1 - (batch // 5) / batch if batch > 4 else 1.0
    size = 1 if case["kind"] == "e4m3" else 2
    rows = batch * nodes * case["heads"]
    own_keys = case["history"] * 5 / 8 + nodes * 3 / 4
    cached = case["shared"] + batch * live * own_keys
    return {"bytes": 2.0 * size * case["kv_heads"] * cached * DIM + 4.0 * rows * DIM + 4.0 * rows * case["lse"]
            + 4.0 * batch * (nodes * -(-nodes // 32) + cached / batch / PAGE),
            "flops": 4.0 * rows * live * 0.75 * (case["shared"] + case["history"] * 5 / 8) * DIM}


def _angles(positions: np.ndarray, case: dict) -> np.ndarray:
    """positions [n] or [n, axes] -> angles [n, pairs] in 64 bits, from the definition."""

    axes, pairs = case.get("axes", 1), case["rotary"] // 2
    positions = positions.reshape(len(positions), -1).astype(np.float64)
    angles = np.empty((len(positions), pairs))
    for k in range(pairs):
        axis, i = divmod(k, pairs // axes)
        angles[:, k] = positions[:, axis] * case["base"] ** (-i / (pairs // axes))
    return angles


def _exactly_turned(x: torch.Tensor, positions: torch.Tensor, case: dict) -> torch.Tensor:
    """x [n, heads, dim]: each pair as a complex number times e^(i angle), in 64 bits."""

    pairs = case["rotary"] // 2
    out = x.double().clone()
    if pairs == 0:
        return out
    angle = torch.from_numpy(_angles(positions.cpu().numpy(), case)).to(x.device)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    first = slice(0, 2 * pairs, 2) if case["interleaved"] else slice(0, pairs)
    second = slice(1, 2 * pairs, 2) if case["interleaved"] else slice(pairs, 2 * pairs)
    z = torch.complex(out[..., first].clone(), out[..., second].clone()) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case: dict, seed: int) -> object:
    if case["op"] == "tree":  # whole numbers only
        return None
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exactly_turned(s["x"], s["positions"], case)
    lengths, table = s["lengths"].cpu().numpy(), s["table"].cpu().numpy()

    def places(b: int, rows: np.ndarray) -> torch.Tensor:
        return torch.from_numpy(table[b, rows // PAGE] * PAGE + rows % PAGE).cuda().long()

    if case["op"] == "keep":
        pools = s["pools"].double()
        for b in range(case["batch"]):
            path = s["path"][b].cpu().numpy()
            path = path[path >= 0].astype(np.int64)
            new = pools[:, :, places(b, lengths[b] + path)].clone()
            pools[:, :, places(b, lengths[b] + np.arange(len(path)))] = new
        return {"pools": pools, "lengths": None}
    counts = s["counts"].cpu().numpy()
    if case["op"] == "append":
        out = {"k": s["k"].double(), "v": s["v"].double()}
        if case["heads"]:
            out["query"] = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
        for b in range(case["batch"]):
            n = int(counts[b])
            at = places(b, lengths[b] + np.arange(n))
            key = _exactly_turned(s["key"][b, :n], s["positions"][b, :n], case)
            for name, new in (("k", key), ("v", s["value"][b, :n].double())):
                if case["kind"] == "e4m3":
                    new = (new / s[name + "_scale"].double()[:, None]).clamp(-448.0, 448.0)
                out[name][:, at] = new.transpose(0, 1)
            if case["heads"]:
                out["query"][b, :n] = _exactly_turned(s["query"][b, :n], s["positions"][b, :n], case)
        return out
    group = case["heads"] // case["kv_heads"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:-1], float("-inf"), dtype=torch.float64, device="cuda")
    bits = np.unpackbits(s["masks"].cpu().numpy().view(np.uint8), axis=-1, bitorder="little").astype(bool)
    for b in range(case["batch"]):
        n, m = int(lengths[b]), int(counts[b])
        if n + m == 0:
            continue
        at = places(b, np.arange(n + m))
        hidden = torch.zeros(m, n + m, dtype=torch.bool, device="cuda")
        hidden[:, n:] = torch.from_numpy(~bits[b, :m, :m]).cuda()
        for g in range(case["kv_heads"]):
            k, v = (s[name][g].view(torch.uint8).view(-1, DIM * s[name].element_size())[at].view(s[name].dtype).double()
                    for name in ("k", "v"))
            if case["kind"] == "e4m3":
                k, v = k * s["k_scale"][g].double(), v * s["v_scale"][g].double()
            q = s["query"][b, :m, g * group:(g + 1) * group].double().transpose(0, 1)
            x = (q @ k.T / math.sqrt(DIM)).masked_fill(hidden, float("-inf"))
            lse[b, :m, g * group:(g + 1) * group] = torch.logsumexp(x, -1).T
            out[b, :m, g * group:(g + 1) * group] = (torch.softmax(x, -1) @ v).transpose(0, 1)
    return {"out": out, "lse": lse} if case["lse"] else {"out": out}
