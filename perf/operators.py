"""Workloads of the branch operators: several continuations ("branches") of one stream that share
its clean history page by page.

The operators are the attention of every branch's new rows over a paged KV cache whose leading
pages all branches share, and the page bookkeeping around it: forking branches off a sequence
(sharing its whole pages and copying its last partial one, or copying everything), releasing
branches, and compacting a pool.

``run`` computes a pass either in plain torch operations in 32 bits (``own`` false) or through the
framework's entry points in ``h3sa.branches`` (``own`` true). ``exact`` is the definition in 64
bits, written apart from both.
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
DIM = 128  # head dimension
ROOT = Path(__file__).resolve().parents[1]


def listed() -> list[dict]:
    return [
        # Two continuations of a short stream, one new token each, three local heads (an eighth
        # of 24): the smallest call, where launches and latency are everything.
        dict(name="attend_two_streams", op="attend", batch=2, rows=1, heads=3, kv_heads=3,
             shared=256, own=57, kind="bf16", causal=False, lse=False),
        # Nine branches with idle slots among them, grouped heads, an e4m3 cache, short history.
        dict(name="attend_e4m3_idle_slots", op="attend", batch=9, rows=1, heads=14, kv_heads=2,
             shared=1152, own=301, kind="e4m3", causal=False, lse=True),
        # Four drafted tokens of each of 24 branches verified at once over a shared document.
        dict(name="attend_drafts", op="attend", batch=24, rows=4, heads=32, kv_heads=8,
             shared=8192, own=700, kind="bf16", causal=True, lse=True),
        # One token each over a very long shared history held in e4m3: bound by reading it once.
        dict(name="attend_e4m3_long_history", op="attend", batch=12, rows=1, heads=40, kv_heads=8,
             shared=98304, own=2100, kind="e4m3", causal=False, lse=False),
        # Whole chunks of three branches (odd row count) over the history: bound by arithmetic.
        dict(name="attend_chunks", op="attend", batch=3, rows=1211, heads=24, kv_heads=24,
             shared=13312, own=2400, kind="bf16", causal=False, lse=False),
        # Two branches off a short sequence in one layer: latency again.
        dict(name="fork_two", op="fork", tensors=2, heads=3, pages=64, sequences=4, width=12,
             children=2, reserve=1, private=False),
        # Sixteen branches over fifty layers (K and V of each), room for a chunk reserved.
        dict(name="fork_all_layers", op="fork", tensors=100, heads=3, pages=240, sequences=6,
             width=40, children=16, reserve=300, private=False),
        # Five private copies of whole sequences over fifty layers: bound by the copy.
        dict(name="fork_private", op="fork", tensors=100, heads=3, pages=300, sequences=6,
             width=40, children=5, reserve=0, private=True),
        # A small pool of one layer, half of it live.
        dict(name="compact_one_layer", op="compact", tensors=2, heads=3, pages=96, sequences=5,
             width=16),
        # The same after many branches came and went, over fifty layers.
        dict(name="compact_all_layers", op="compact", tensors=100, heads=3, pages=256,
             sequences=24, width=40),
        # Two of a few branches end.
        dict(name="free_few", op="free", pages=512, sequences=8, width=64),
        # Many branches of a large pool end at once.
        dict(name="free_many", op="free", pages=40000, sequences=256, width=1000),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(["attend", "attend", "attend", "fork", "compact", "free"])
    if op == "attend":
        while True:
            kv_heads = rng.choice([1, 2, 3, 4, 8, 14, 24])
            group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
            case = dict(op=op, batch=_log(rng, 1, 100), rows=_log(rng, 1, 2000) if rng.random() < 0.4 else rng.randint(1, 9),
                        heads=kv_heads * group, kv_heads=kv_heads,
                        shared=PAGE * (_log(rng, 1, 800) if rng.random() < 0.9 else 0),
                        own=_log(rng, 1, 3000), kind=rng.choice(["bf16", "bf16", "e4m3"]),
                        causal=rng.random() < 0.5, lse=rng.random() < 0.3)
            keys = case["shared"] + case["own"]
            scores = case["batch"] * case["rows"] * case["heads"] * keys
            cells = kv_heads * (case["shared"] + case["batch"] * (case["own"] + PAGE))
            # no more arithmetic, and no more cache, than the largest listed calls
            if scores <= 1.2e9 and cells <= 1.2e6 and scores >= 1e3:
                return case
    sequences = _log(rng, 1, 30)
    width = rng.randint(3, 48)
    layers = _log(rng, 1, 50)
    heads = rng.choice([1, 2, 3, 6, 8, 24])
    if op == "fork":
        children = _log(rng, 1, 40)
        private = rng.random() < 0.3
        reserve = _log(rng, 1, 700) if rng.random() < 0.7 else 0
        pages = sequences * width + children * (1 + -(-reserve // PAGE) + (width if private else 0)) + rng.randint(0, 40)
        while layers > 1 and 2 * layers * heads * pages > 90000:
            layers //= 2
        while 2 * layers * heads * pages > 90000:
            heads = max(1, heads // 2)
            pages = min(pages, 45000)
        return dict(op=op, tensors=2 * layers, heads=heads, pages=pages, sequences=sequences,
                    width=width + -(-reserve // PAGE) + 1, children=children, reserve=reserve,
                    private=private)
    if op == "compact":
        pages = max(8, int(sequences * width * rng.uniform(0.6, 1.5)))
        while layers > 1 and 2 * layers * heads * pages > 76000:
            layers //= 2
        while 2 * layers * heads * pages > 76000:
            heads = max(1, heads // 2)
        return dict(op=op, tensors=2 * layers, heads=heads, pages=pages, sequences=sequences,
                    width=width)
    sequences = _log(rng, 1, 256)
    width = _log(rng, 4, 1000)
    return dict(op=op, pages=max(16, min(40000, int(sequences * width * 0.5))), sequences=sequences,
                width=width)


# ------------------------------------------------------------------------------------ inputs


def _ledger(rs: np.random.RandomState, sequences: int, width: int, pages: int, spare: int,
            fill: float) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """A pool's bookkeeping in use: sequences in families of up to four that share leading pages
    and have pages of their own after them, page numbers scattered over the pool. Returns the
    table [sequences, width] (-1 where no page is held), the lengths and the reference counts."""

    table = np.full((sequences, width), -1, np.int64)
    lengths = np.zeros(sequences, np.int64)
    ids = rs.permutation(pages)
    room = min(pages - spare, int(pages * fill))
    at = 0
    common: np.ndarray = ids[:0]
    for s in range(sequences):
        if s % 4 == 0:
            k = min(rs.randint(0, max(1, width // 2) + 1), max(0, room - at))
            common = ids[at:at + k]
            at += k
        k = min(rs.randint(0, width - len(common) + 1), max(0, room - at))
        held = np.concatenate([common, ids[at:at + k]])
        at += k
        table[s, :len(held)] = held
        if len(held):
            lengths[s] = (len(held) - 1) * PAGE + (rs.randint(1, PAGE + 1) if k else PAGE)
    refs = np.bincount(table[table >= 0], minlength=pages)
    return table, lengths, refs


def _dev(a: np.ndarray, dtype: torch.dtype = torch.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def _pool(gen: torch.Generator, shape: tuple[int, ...]) -> torch.Tensor:
    """Cache rows as a model leaves them: unit-variance bf16."""

    out = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
    return out.normal_(generator=gen)


def prepare(case: dict, seed: int) -> dict:
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=case)
    if case["op"] == "attend":
        batch, shared = case["batch"], case["shared"] // PAGE
        extra = rs.randint(0, case["own"] + 1, batch)
        extra[rs.randint(batch)] = case["own"]
        lengths = shared * PAGE + extra
        if batch > 4:
            lengths[rs.randint(batch, size=batch // 5)] = 0  # slots without a branch
        held = -(-lengths // PAGE)
        width = shared + -(-case["own"] // PAGE)
        pages = shared + int(np.maximum(held - shared, 0).sum()) + 3
        ids = rs.permutation(pages)
        table = np.full((batch, max(1, width)), -1, np.int64)
        at = shared
        for b in range(batch):
            if lengths[b]:
                k = held[b] - shared
                table[b, :shared] = ids[:shared]
                table[b, shared:held[b]] = ids[at:at + k]
                at += k
        shape = (case["kv_heads"], pages * PAGE, DIM)
        key, value = _pool(gen, shape), _pool(gen, shape)
        query = torch.empty(batch, case["rows"], case["heads"], DIM, device="cuda")
        state["query"] = query.normal_(0.0, 1.5, generator=gen).bfloat16()
        if case["kind"] == "e4m3":
            for name, t in (("k", key), ("v", value)):
                scale = t.abs().amax(dim=(1, 2)).float() / 448.0
                state[name + "_scale"] = scale
                state[name] = (t.float() / scale[:, None, None]).to(torch.float8_e4m3fn)
        else:
            state["k"], state["v"] = key, value
        state["table"], state["lengths"] = _dev(table), _dev(lengths)
        return state
    spare, fill = 0, 1.0
    if case["op"] == "fork":
        fresh = 1 + -(-case["reserve"] // PAGE)
        width = case["width"] - fresh
        spare = case["children"] * (fresh + (width if case["private"] else 0))
    else:
        width = case["width"]
        fill = 0.55 if case["op"] == "compact" else 1.0
    table, lengths, refs = _ledger(rs, case["sequences"], width, case["pages"], spare, fill)
    table = np.pad(table, ((0, 0), (0, case["width"] - width)), constant_values=-1)
    state["table"], state["lengths"], state["refs"] = _dev(table), _dev(lengths), _dev(refs)
    if case["op"] == "free":
        state["release"] = _dev(rs.rand(case["sequences"]) < 0.4, torch.bool)
        return state
    state["pools"] = _pool(gen, (case["tensors"], case["heads"], case["pages"] * PAGE, DIM))
    if case["op"] == "fork":
        parents = rs.randint(0, case["sequences"], case["children"])
        parents[rs.rand(case["children"]) < 0.1] = -1  # a branch that starts empty
        state["parents"] = _dev(parents)
    return state


# ------------------------------------------------------------------------------ plain forms


def _attend_plain(s: dict) -> dict:
    c = s["case"]
    batch, rows, heads, kv = c["batch"], c["rows"], c["heads"], c["kv_heads"]
    group, shared = heads // kv, c["shared"] // PAGE
    width = s["table"].shape[1]
    k = s["k"].view(kv, -1, PAGE, DIM)
    v = s["v"].view(kv, -1, PAGE, DIM)
    lengths = s["lengths"].long()
    table = s["table"].long()
    scale = DIM ** -0.5

    def rows_of(pool: torch.Tensor, pages: torch.Tensor, name: str) -> torch.Tensor:
        x = pool.view(torch.uint8)[:, pages].view(pool.dtype).float()
        return x * s[name][:, *([None] * (x.ndim - 1))] if name in s else x

    # [kv, batch, rows * group, dim]
    q = s["query"].float().view(batch, rows, kv, group, DIM).permute(2, 0, 1, 3, 4)
    q = q.reshape(kv, batch, rows * group, DIM).contiguous() * scale
    first = table[lengths.argmax()]
    kp = rows_of(k, first[:shared].clamp(min=0), "k_scale").reshape(kv, shared * PAGE, DIM)
    vp = rows_of(v, first[:shared].clamp(min=0), "v_scale").reshape(kv, shared * PAGE, DIM)
    tail = (width - shared) * PAGE
    ks = rows_of(k, table[:, shared:].clamp(min=0), "k_scale").reshape(kv, batch, tail, DIM)
    vs = rows_of(v, table[:, shared:].clamp(min=0), "v_scale").reshape(kv, batch, tail, DIM)
    at = torch.arange(width * PAGE, device=q.device)
    vs = torch.where((at[shared * PAGE:] < lengths[:, None])[None, :, :, None], vs, 0.0)
    limit = lengths[:, None] - (rows - 1 - torch.arange(rows, device=q.device) if c["causal"]
                                else torch.zeros(rows, dtype=torch.long, device=q.device))
    seen = (at < limit[:, :, None]).repeat_interleave(group, 1)  # [batch, rows * group, keys]
    low = torch.tensor(float("-inf"), device=q.device)
    sp = torch.matmul(q.view(kv, -1, DIM), kp.transpose(1, 2)).view(kv, batch, rows * group, -1)
    sp = torch.where(seen[:, :, :shared * PAGE], sp, low)
    ss = torch.where(seen[:, :, shared * PAGE:], torch.matmul(q, ks.transpose(2, 3)), low)
    parts = torch.cat((sp, ss), -1)
    top = parts.amax(-1, keepdim=True)
    base = torch.where(top.isinf(), 0.0, top)
    p = torch.exp(parts - base)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :shared * PAGE].reshape(kv, batch * rows * group, shared * PAGE), vp).view(q.shape)
    o = o + torch.matmul(p[..., shared * PAGE:], vs)
    o = torch.where(total > 0, o / total, 0.0)
    back = lambda t: t.view(kv, batch, rows, group, -1).permute(1, 2, 0, 3, 4).reshape(batch, rows, heads, -1)  # noqa: E731
    out = {"out": back(o).bfloat16()}
    if c["lse"]:
        out["lse"] = back(base + torch.log(total)).squeeze(-1)
    return out


def _fork_plain(s: dict) -> dict:
    c = s["case"]
    table, lengths, refs = s["table"].long(), s["lengths"].long(), s["refs"].long()
    parents = s["parents"].long()
    known = parents >= 0
    n = torch.where(known, lengths[parents.clamp(min=0)], 0)
    mine = table[parents.clamp(min=0)]
    held = -(-n // PAGE)
    kept = torch.zeros_like(n) if c["private"] else n // PAGE  # pages shared with the parent
    need = -(-(n + c["reserve"]) // PAGE)
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)  # free pages first, in order
    start = torch.cumsum(need - kept, 0) - (need - kept)
    j = torch.arange(c["width"], device=table.device)
    fresh = free[(start[:, None] + j - kept[:, None]).clamp(0, c["pages"] - 1)]
    child = torch.where(j < kept[:, None], mine, torch.where(j < need[:, None], fresh, -1))
    ones = (child >= 0).long().view(-1)
    refs = refs.scatter_add(0, child.clamp(min=0).view(-1), ones)
    # whole pages are written back row by row where the parent has a row; entries without a copy
    # rewrite a page that is in use with itself
    copied = (j >= kept[:, None]) & (j < held[:, None])
    idle = s["refs"].argmax()
    src = torch.where(copied, mine, idle).view(-1)
    dst = torch.where(copied, child, idle).view(-1)
    has = (j[:, None] * PAGE + torch.arange(PAGE, device=j.device)) < n[:, None, None]
    if not c["private"]:  # at most one page of a branch is copied, the one at `kept`
        pick = kept.clamp(max=c["width"] - 1)[:, None]
        src = src.view(child.shape).gather(1, pick).view(-1)
        dst = dst.view(child.shape).gather(1, pick).view(-1)
        has = has[torch.arange(len(n), device=j.device), pick.view(-1)]
    pool = s["pools"].view(c["tensors"], c["heads"], c["pages"], PAGE, DIM)
    pool[:, :, dst] = torch.where(has.view(-1, PAGE, 1), pool[:, :, src], pool[:, :, dst])
    return {"table": child.int(), "lengths": n.int(), "refs": refs.int(), "pools": s["pools"]}


def _compact_plain(s: dict) -> dict:
    c = s["case"]
    table, refs = s["table"].long(), s["refs"].long()
    at = torch.arange(c["pages"], device=table.device)
    live = refs > 0
    count = live.sum()
    hole = ~live & (at < count)  # the i-th hole takes the i-th live page past the end
    mover = live & (at >= count)
    holes = torch.argsort((~hole).to(torch.int8), stable=True)
    rank = torch.cumsum(mover.long(), 0) - 1
    to = torch.where(mover, holes[rank.clamp(min=0)], at)
    table = torch.where(table >= 0, to[table.clamp(min=0)], -1)
    moved = torch.zeros_like(refs).scatter_add(0, to, torch.where(live, refs, 0))
    pool = s["pools"].view(c["tensors"], c["heads"], c["pages"], PAGE, DIM)
    half = c["pages"] // 2 + 1  # no more pages than that can move
    movers = torch.argsort((~mover).to(torch.int8), stable=True)[:half]
    still = ~mover[movers]  # entries past the last mover: rewrite a page with itself
    last = at[-1]  # a hole is never the last page
    src = torch.where(still & hole[movers], last, movers)  # ... but no page that is being filled
    dst = torch.where(still, src, to[movers])
    pool[:, :, dst] = pool[:, :, src]
    return {"table": table.int(), "refs": moved.int(), "live": count.int().view(1),
            "pools": s["pools"]}


def _free_plain(s: dict) -> dict:
    table, refs, gone = s["table"].long(), s["refs"].long(), s["release"]
    drop = ((table >= 0) & gone[:, None]).long().view(-1)
    refs = refs.scatter_add(0, table.clamp(min=0).view(-1), -drop)
    table = torch.where(gone[:, None], -1, table)
    return {"table": table.int(), "lengths": torch.where(gone, 0, s["lengths"]),
            "refs": refs.int()}


# ------------------------------------------------------------------------ the framework's own


def _branches():
    at = str(ROOT / "taomate-h3_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import h3sa.branches

    return h3sa.branches


def _own(s: dict) -> dict:
    c = s["case"]
    ops = _branches()
    if c["op"] == "attend":
        lse = torch.empty(c["batch"], c["rows"], c["heads"], device="cuda") if c["lse"] else None
        out = ops.shared_prefix_attention(s["query"], s["k"], s["v"], s["table"], s["lengths"],
                                          c["shared"], DIM ** -0.5, causal=c["causal"],
                                          k_scale=s.get("k_scale"), v_scale=s.get("v_scale"),
                                          lse=lse)
        return {"out": out} if lse is None else {"out": out, "lse": lse}
    if c["op"] == "fork":
        table, lengths, refs = ops.fork_pages(s["pools"], s["table"], s["lengths"], s["refs"],
                                              s["parents"], reserve_rows=c["reserve"],
                                              private=c["private"])
        return {"table": table, "lengths": lengths, "refs": refs, "pools": s["pools"]}
    if c["op"] == "compact":
        table, refs, live = ops.compact_pages(s["pools"], s["table"], s["refs"])
        return {"table": table, "refs": refs, "live": live, "pools": s["pools"]}
    table, lengths, refs = ops.free_pages(s["table"], s["lengths"], s["refs"], s["release"])
    return {"table": table, "lengths": lengths, "refs": refs}


def run(state: dict) -> dict:
    if own:
        return _own(state)
    plain = {"attend": _attend_plain, "fork": _fork_plain, "compact": _compact_plain,
             "free": _free_plain}
    return plain[state["case"]["op"]](state)


# ---------------------------------------------------------------------------- cost and truth


def _lengths(case: dict) -> np.ndarray:
    """Mean lengths of the drawn inputs (their exact ones depend on the seed)."""

    full = case["shared"] + case["own"] / 2
    idle = (case["batch"] // 5) / case["batch"] if case["batch"] > 4 else 0.0
    return np.full(case["batch"], full * (1 - idle))


def work(case: dict) -> dict:
    if case["op"] == "attend":
        size = 1 if case["kind"] == "e4m3" else 2
        rows = case["batch"] * case["rows"] * case["heads"]
        cached = case["shared"] + case["batch"] * case["own"] / 2
        width = case["shared"] // PAGE + -(-case["own"] // PAGE)
        moved = 2 * size * case["kv_heads"] * cached * DIM + 4 * rows * DIM + 4 * rows * case["lse"]
        seen = float(_lengths(case).mean()) - (case["rows"] - 1) / 2 * case["causal"]
        return {"bytes": moved + 4 * case["batch"] * (width + 1),
                "flops": 4.0 * rows * max(1.0, seen) * DIM}
    cells = case["sequences"] * case["width"]
    if case["op"] == "free":
        return {"bytes": 4.0 * (2 * cells + 2 * case["sequences"] + 2 * case["pages"])
                + case["sequences"], "flops": 0.0}
    plane = 2 * case["tensors"] * case["heads"] * DIM * 2  # a row read and written everywhere
    if case["op"] == "compact":
        live = 0.55 * case["pages"]
        return {"bytes": plane * PAGE * 0.45 * live + 4.0 * (2 * cells + 2 * case["pages"]),
                "flops": 0.0}
    mean = max(1, case["width"] - 1 - -(-case["reserve"] // PAGE)) * PAGE * 0.6
    rows = case["children"] * 0.9 * (mean if case["private"] else PAGE / 2)
    return {"bytes": plane * rows + 4.0 * (2 * case["children"] * case["width"]
                                           + 2 * case["pages"]), "flops": 0.0}


def _attend_exact(s: dict) -> dict:
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:-1], float("-inf"), dtype=torch.float64, device="cuda")
    table, lengths = s["table"].cpu().numpy(), s["lengths"].cpu().numpy()
    for b in range(c["batch"]):
        n = int(lengths[b])
        if n == 0:
            continue
        at = torch.from_numpy((table[b, np.arange(n) // PAGE] * PAGE + np.arange(n) % PAGE)).cuda()
        last = torch.arange(c["rows"], device="cuda") - (c["rows"] - 1) if c["causal"] else torch.zeros(c["rows"], device="cuda")
        hidden = torch.arange(n, device="cuda")[None] >= (n + last)[:, None]
        for h in range(c["heads"]):
            g = h // group
            k = s["k"][g].view(torch.uint8)[at].view(s["k"].dtype).double()
            v = s["v"][g].view(torch.uint8)[at].view(s["v"].dtype).double()
            if c["kind"] == "e4m3":
                k, v = k * s["k_scale"][g].double(), v * s["v_scale"][g].double()
            x = (s["query"][b, :, h].double() @ k.T) / math.sqrt(DIM)
            x.masked_fill_(hidden, float("-inf"))
            lse[b, :, h] = torch.logsumexp(x, -1)
            out[b, :, h] = torch.softmax(x, -1).nan_to_num(0.0) @ v
    return {"out": out, "lse": lse} if c["lse"] else {"out": out}


def exact(case: dict, seed: int) -> dict | None:
    if case["op"] == "free":  # whole numbers only
        return None
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _attend_exact(s)
    pool = s["pools"].double().view(case["tensors"], case["heads"], case["pages"], PAGE, DIM)
    table, refs = s["table"].cpu().numpy(), s["refs"].cpu().numpy()
    if case["op"] == "compact":
        live = np.flatnonzero(refs)
        holes = np.setdiff1d(np.arange(len(live)), live)
        for src, dst in zip(live[live >= len(live)], holes):
            pool[:, :, dst] = pool[:, :, src]
        return {"table": None, "refs": None, "live": None, "pools": pool.view(s["pools"].shape)}
    free = iter(np.flatnonzero(refs == 0))
    for p in s["parents"].cpu().numpy():
        n = int(s["lengths"][p]) if p >= 0 else 0
        kept = 0 if case["private"] else n // PAGE
        for page in range(kept, -(-(n + case["reserve"]) // PAGE)):
            dst, filled = next(free), min(PAGE, n - page * PAGE)
            if filled > 0:
                pool[:, :, dst, :filled] = pool[:, :, table[p, page], :filled]
    return {"table": None, "lengths": None, "refs": None, "pools": pool.view(s["pools"].shape)}
