"""Drafted trees and rotary positions, restated in plain numpy / torch on the CPU in 64 bits.

There is no counterpart in the reference.
"""

from __future__ import annotations

import numpy as np
import torch

PAGE = 128


def ancestors(parents: np.ndarray, counts: np.ndarray) -> np.ndarray:
    """bool [batch, nodes, nodes]: whether a node is another or below it; a parent that is none makes a root."""

    batch, nodes = parents.shape
    sees = np.zeros((batch, nodes, nodes), bool)
    for b in range(batch):
        for i in range(max(0, min(nodes, int(counts[b])))):
            p = int(parents[b, i])
            if 0 <= p < i:
                sees[b, i] = sees[b, p]
            sees[b, i, i] = True
    return sees


def words(sees: np.ndarray) -> np.ndarray:
    """bool [..., n] as int32 [..., ceil(n / 32)], the lowest bit first."""

    n = sees.shape[-1]
    out = np.zeros((*sees.shape[:-1], -(-n // 32)), np.uint32)
    for j in range(n):
        out[..., j // 32] |= sees[..., j].astype(np.uint32) << np.uint32(j % 32)
    return out.view(np.int32)


def rotate(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, interleaved: bool = False,
           factor: float = 1.0) -> torch.Tensor:
    """x [..., heads, dim] in 64 bits; positions [..., axes], frequencies [axes, pairs of an axis]."""

    axes, per = frequencies.shape
    pairs = axes * per
    out = x.double().clone()
    for k in range(pairs):
        a = positions[..., k // per].double() * frequencies[k // per, k % per]
        i, j = (2 * k, 2 * k + 1) if interleaved else (k, k + pairs)
        u, v = x[..., i].double(), x[..., j].double()
        c, s = torch.cos(a)[..., None] * factor, torch.sin(a)[..., None] * factor
        out[..., i], out[..., j] = u * c - v * s, u * s + v * c
    return out


def places(table: np.ndarray, b: int, rows: np.ndarray) -> torch.Tensor:
    rows = np.asarray(rows, np.int64)
    return torch.from_numpy(table[b, rows // PAGE].astype(np.int64) * PAGE + rows % PAGE)


def keep(pool: torch.Tensor, table: np.ndarray, lengths: np.ndarray, path: np.ndarray):
    """pool [..., pages * 128, d] -> (pool, lengths); paths are taken as they are."""

    out, kept = pool.clone(), lengths.copy()
    for b in range(len(lengths)):
        steps = list(path[b])
        steps = steps[:next((k for k, n in enumerate(steps) if n < 0), len(steps))]
        if steps:
            out[..., places(table, b, lengths[b] + np.arange(len(steps))), :] = \
                pool[..., places(table, b, lengths[b] + np.array(steps)), :]
        kept[b] += len(steps)
    return out, kept


def attention(query: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, table: np.ndarray,
              lengths: np.ndarray, counts: np.ndarray, sees: np.ndarray, scale: float,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None):
    """float64 (out [B, n, H, d], lse [B, n, H], sum of p |v|, largest p times sum of |v|): the last two bound
    what rounding p can change. sees: bool [B, n, n]."""

    batch, rows, heads, _ = query.shape
    group = heads // key_pool.shape[0]
    out = torch.zeros(query.shape, dtype=torch.float64)
    lse = torch.full((batch, rows, heads), float("-inf"), dtype=torch.float64)
    spread, peak = torch.zeros_like(out), torch.zeros_like(out)
    for b in range(batch):
        n, m = int(lengths[b]), int(counts[b])
        if m == 0 or n + m == 0:
            continue
        at = places(table, b, np.arange(n + m))
        for h in range(heads):
            k, v = key_pool[h // group].double()[at], value_pool[h // group].double()[at]
            if k_scale is not None:
                k, v = k * k_scale[h // group].double(), v * v_scale[h // group].double()
            for i in range(m):
                seen = np.concatenate([np.ones(n, bool), sees[b, i, :m]])
                if not seen.any():
                    continue
                where = torch.from_numpy(np.flatnonzero(seen))
                x = k[where] @ query[b, i, h].double() * scale
                lse[b, i, h] = torch.logsumexp(x, 0)
                p = torch.exp(x - lse[b, i, h])
                out[b, i, h] = p @ v[where]
                spread[b, i, h] = p @ v[where].abs()
                peak[b, i, h] = p.max() * v[where].abs().sum(0)
    return out, lse, spread, peak
