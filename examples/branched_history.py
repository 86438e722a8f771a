"""Candidate continuations of one clean history, the branch operators together.

A stack of attention layers holds one stream's clean KV history in pages. ``branches`` candidates
continue it: each forks the history (whole pages are held together, only the partial last page is
copied), writes ``rows`` new rows a step behind it in every layer and attends from them, the
history being read once for all candidates. After every round of steps one candidate is kept, the
others are freed, the pages in use move to the front of the pools, and the next round forks what
is left. ``--check`` recomputes each attention from dense rows in fp64.

    PYTHONPATH=taomate-h3_b200 python examples/branched_history.py --branches 4 --rows 16 --check
"""

from __future__ import annotations

import argparse
import math

import torch

from h3sa.branches import compact_pages, fork_pages, free_pages, shared_prefix_attention
from h3sa.cache import PagedLayerKV
from h3sa.kernels import HEAD_DIM, PAGE_ROWS, kv_copy_rows


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """fp64 attention of the last rows of a sequence: q [n, heads, 128], k and v [rows, kv_heads, 128]."""

    n, heads, _ = q.shape
    group = heads // k.shape[1]
    k, v = (t.double().repeat_interleave(group, dim=1) for t in (k, v))
    x = torch.einsum("nhd,shd->hns", q.double(), k) / math.sqrt(HEAD_DIM)
    first = k.shape[0] - n  # row i sees keys up to itself
    hidden = torch.arange(k.shape[0], device=q.device)[None, :] > first + torch.arange(n, device=q.device)[:, None]
    return torch.einsum("hns,shd->nhd", x.masked_fill(hidden, -math.inf).softmax(dim=-1), v)


class Branches:
    """Sequences over the pools of all layers: a ledger on the device, lengths known to the host."""

    def __init__(self, layers: list[PagedLayerKV], rows: int) -> None:
        device = layers[0].device
        pages = (rows + PAGE_ROWS - 1) // PAGE_ROWS
        if any(layer.pages != layers[0].pages or layer.capacity != layers[0].capacity for layer in layers):
            raise RuntimeError("the layers' histories must lie in the same pages")
        self.pools = [t for layer in layers for t in (layer.key, layer.value)]
        self.refs = torch.zeros(layers[0].capacity, dtype=torch.int32, device=device)
        self.table = torch.full((1, layers[0].capacity), -1, dtype=torch.int32, device=device)
        self.table[0, :pages] = layers[0].table[:pages]
        self.refs[self.table[0, :pages].long()] = 1
        self.lengths = torch.tensor([rows], dtype=torch.int32, device=device)
        self.rows, self.shared = rows, 0  # every sequence's length; rows in pages that all hold
        self.error = torch.zeros(1, dtype=torch.int32, device=device)

    def fork(self, count: int, reserve: int) -> None:
        """``count`` branches of sequence 0, which itself ends; each has pages for ``reserve`` more rows."""

        parents = torch.zeros(count, dtype=torch.int32, device=self.refs.device)
        table, lengths, refs = fork_pages(self.pools, self.table, self.lengths, self.refs, parents,
                                          reserve_rows=reserve, device_error=self.error)
        ended = torch.ones(1, dtype=torch.bool, device=refs.device)
        _, _, self.refs = free_pages(self.table, self.lengths, refs, ended, device_error=self.error)
        self.table, self.lengths = table, lengths
        self.shared = self.rows // PAGE_ROWS * PAGE_ROWS

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """New rows ``[branches, n, kv_heads, 128]`` of one layer behind every branch."""

        for b in range(key.shape[0]):
            kv_copy_rows([key[b], value[b]], self.pools[2 * layer:2 * layer + 2], count=key.shape[1],
                         dst_table=self.table[b], dst_start=self.rows, device_error=self.error)

    def advance(self, rows: int) -> None:
        self.rows += rows
        self.lengths = self.lengths + rows

    def attend(self, layer: int, query: torch.Tensor, rows: int) -> torch.Tensor:
        """The last rows' attention; ``rows`` of them were appended and not yet counted."""

        return shared_prefix_attention(query, *self.pools[2 * layer:2 * layer + 2], self.table,
                                       self.lengths + rows, self.shared, HEAD_DIM ** -0.5, causal=True,
                                       device_error=self.error)

    def keep(self, branch: int) -> torch.Tensor:
        """End all branches but one and close the gaps; returns the pages in use."""

        release = torch.ones(self.table.shape[0], dtype=torch.bool, device=self.refs.device)
        release[branch] = False
        table, lengths, refs = free_pages(self.table, self.lengths, self.refs, release, device_error=self.error)
        table, self.refs, live = compact_pages(self.pools, table, refs, device_error=self.error)
        self.table, self.lengths = table[branch:branch + 1].clone(), lengths[branch:branch + 1].clone()
        return live


def run(layers: int = 4, heads: int = 8, kv_heads: int = 2, history: int = 1000, branches: int = 4,
        rows: int = 16, steps: int = 3, rounds: int = 3, check: bool = False, seed: int = 0) -> float:
    """Returns the largest error of a checked output relative to the largest value (0 unchecked)."""

    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)

    def draw(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device=device).to(torch.bfloat16)

    most = history + rounds * steps * rows
    pages = most // PAGE_ROWS + 1 + branches * (steps * rows // PAGE_ROWS + 2)
    clean = [PagedLayerKV(kv_heads, HEAD_DIM, torch.bfloat16, device, initial_pages=pages) for _ in range(layers)]
    dense = [[draw(history, kv_heads, HEAD_DIM) for _ in range(2)] for _ in range(layers)]
    for layer, (key, value) in zip(clean, dense):
        layer.write(key, value, start=0, count=history)
    held = Branches(clean, history)
    worst = 0.0
    for _ in range(rounds):
        held.fork(branches, steps * rows)
        ends = [[[key, value] for _ in range(branches)] for key, value in dense] if check else []
        scores = torch.zeros(branches, device=device)
        for _ in range(steps):
            for layer in range(layers):
                query = draw(branches, rows, heads, HEAD_DIM)
                key, value = (draw(branches, rows, kv_heads, HEAD_DIM) for _ in range(2))
                held.append(layer, key, value)
                out = held.attend(layer, query, rows)
                scores += out.float().square().mean(dim=(1, 2, 3))
                for b in range(branches if check else 0):
                    both = ends[layer][b] = [torch.cat([t, new[b]]) for t, new in zip(ends[layer][b], (key, value))]
                    want = dense_attention(query[b], *both)
                    worst = max(worst, float((out[b] - want).abs().max() / both[1].abs().max()))
            held.advance(rows)
        best = int(scores.argmax())
        if check:
            dense = [ends[layer][best] for layer in range(layers)]
        live = int(held.keep(best))
        print(f"kept branch {best}: {held.rows} rows in {live} pages, {int(held.refs.count_nonzero())} held")
    if int(held.error):
        raise RuntimeError(f"device error word {int(held.error):#x}")
    return worst


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("layers", 4), ("heads", 8), ("kv-heads", 2), ("history", 1000), ("branches", 4),
                        ("rows", 16), ("steps", 3), ("rounds", 3)):
        parser.add_argument(f"--{name}", type=int, default=value)
    parser.add_argument("--check", action="store_true")
    worst = run(**vars(parser.parse_args()))
    print(f"largest error {worst:.2e} of the largest value")


if __name__ == "__main__":
    main()
