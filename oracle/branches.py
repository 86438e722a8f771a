"""Branches over shared pages, restated in plain numpy / torch on the CPU.

The ledger operations as loops over pages, and attention in 64 bits straight from its definition.
There is no counterpart in the reference.
"""

from __future__ import annotations

import numpy as np
import torch

PAGE = 128


def pages_of(rows: int) -> int:
    return -(-rows // PAGE)


def fork(table: np.ndarray, lengths: np.ndarray, refs: np.ndarray, parents: np.ndarray, *,
         reserve_rows: int = 0, private: bool = False):
    """Returns (child_table, child_lengths, refs, moves): moves are (source, destination, rows)."""

    width = table.shape[1]
    free = list(np.flatnonzero(refs == 0))
    refs = refs.copy()
    child = np.full((len(parents), width), -1, table.dtype)
    child_lengths = np.zeros(len(parents), lengths.dtype)
    moves = []
    for c, p in enumerate(parents):
        n = int(lengths[p]) if p >= 0 else 0
        kept = 0 if private else n // PAGE
        for j in range(pages_of(n + reserve_rows)):
            if j < kept:
                child[c, j] = table[p, j]
                refs[table[p, j]] += 1
                continue
            child[c, j] = free.pop(0)
            refs[child[c, j]] = 1
            if j * PAGE < n:
                moves.append((int(table[p, j]), int(child[c, j]), min(PAGE, n - j * PAGE)))
        child_lengths[c] = n
    return child, child_lengths, refs, moves


def compact(table: np.ndarray, refs: np.ndarray):
    """Returns (table, refs, live, moves)."""

    used = np.flatnonzero(refs > 0)
    live = len(used)
    holes = [p for p in range(live) if refs[p] == 0]
    moves = [(int(src), int(dst), PAGE) for src, dst in zip(used[used >= live], holes)]
    to = np.full(len(refs) + 1, -1, table.dtype)  # the last entry is where -1 points
    to[used[used < live]] = used[used < live]
    out = np.zeros_like(refs)
    out[used[used < live]] = refs[used[used < live]]
    for src, dst, _ in moves:
        to[src] = dst
        out[dst] = refs[src]
    return to[table], out, live, moves


def free(table: np.ndarray, lengths: np.ndarray, refs: np.ndarray, release: np.ndarray):
    table, lengths, refs = table.copy(), lengths.copy(), refs.copy()
    for s in np.flatnonzero(release):
        for page in table[s][table[s] >= 0]:
            refs[page] -= 1
        table[s] = -1
        lengths[s] = 0
    return table, lengths, refs


def copy_rows(pool: torch.Tensor, moves) -> torch.Tensor:
    """The moves applied to pool tensors [..., pages * 128, d]."""

    out = pool.clone()
    for src, dst, rows in moves:
        out[..., dst * PAGE:dst * PAGE + rows, :] = pool[..., src * PAGE:src * PAGE + rows, :]
    return out


def attention(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, table: np.ndarray,
              lengths: np.ndarray, scale: float, *, causal: bool = False,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
    """float64 (out [B, n, H, d], lse [B, n, H], sum of p |v|, largest p times sum of |v|): the
    last two bound what rounding p can change."""

    batch, rows, heads, d = query.shape
    group = heads // key_pool.shape[0]
    out = torch.zeros(query.shape, dtype=torch.float64)
    lse = torch.full((batch, rows, heads), float("-inf"), dtype=torch.float64)
    spread, peak = torch.zeros_like(out), torch.zeros_like(out)
    for b in range(batch):
        n = int(lengths[b])
        at = torch.tensor([int(table[b, j // PAGE]) * PAGE + j % PAGE for j in range(n)], dtype=torch.long)
        for h in range(heads):
            k = key_pool[h // group].double()[at]
            v = value_pool[h // group].double()[at]
            if k_scale is not None:
                k, v = k * k_scale[h // group].double(), v * v_scale[h // group].double()
            for i in range(rows):
                seen = max(0, n - (rows - 1 - i if causal else 0))
                if seen == 0:
                    continue
                x = k[:seen] @ query[b, i, h].double() * scale
                lse[b, i, h] = torch.logsumexp(x, 0)
                p = torch.exp(x - lse[b, i, h])
                out[b, i, h] = p @ v[:seen]
                spread[b, i, h] = p @ v[:seen].abs()
                peak[b, i, h] = p.max() * v[:seen].abs().sum(0)
    return out, lse, spread, peak
