"""Drafted trees over one shared history, the operators of a drafting step together.

``sequences`` continuations fork a clean history of rotated keys, the whole pages of which they hold together. In every step a
tree of rows is proposed behind each of them: its ancestor bits and positions are worked out once, every layer
appends the rows' keys and values to the pages, with keys and queries rotated on the way, and attends from all
rows at once; then the rows of one path of each tree become history in all layers. ``--check`` recomputes each attention from dense
rows in fp64.

    PYTHONPATH=taomate-h3_b200 python examples/drafted_trees.py --sequences 4 --nodes 12 --check
"""

from __future__ import annotations

import argparse
import math

import torch

from h3sa.branches import fork_pages
from h3sa.drafts import append_rows, draft_tree, keep_rows, tree_attention
from h3sa.kernels import HEAD_DIM, PAGE_ROWS
from h3sa.rotary import rotary_frequencies, rotate


def turned(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor) -> torch.Tensor:
    """fp64 rotation of [rows, heads, 128] in halves, rounded to bf16 as a cache holds it."""

    angle = (positions[:, None].double() * frequencies)[:, None]
    pairs = frequencies.numel()
    a, b, rest = x[..., :pairs].double(), x[..., pairs:2 * pairs].double(), x[..., 2 * pairs:].double()
    return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), rest), -1).bfloat16()


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """fp64 attention of one row: q [heads, 128], k and v [rows, kv_heads, 128]."""

    group = q.shape[0] // k.shape[1]
    k, v = (t.double().repeat_interleave(group, dim=1) for t in (k, v))
    p = (torch.einsum("hd,shd->hs", q.double(), k) / math.sqrt(HEAD_DIM)).softmax(dim=-1)
    return torch.einsum("hs,shd->hd", p, v)


def random_trees(sequences: int, nodes: int, g: torch.Generator) -> tuple[list[list[int]], list[int]]:
    """Parents of every row (in front of it, -1 for the root) and the rows that each sequence proposes."""

    counts = [int(torch.randint(1, nodes + 1, (), generator=g)) for _ in range(sequences)]
    parents = [[-1] + [int(torch.randint(max(0, i - 4), i, (), generator=g)) for i in range(1, nodes)] for _ in range(sequences)]
    return parents, counts


def path_to(parents: list[int], leaf: int) -> list[int]:
    path = [leaf]
    while parents[path[-1]] >= 0:
        path.append(parents[path[-1]])
    return path[::-1]


def run(layers: int = 3, heads: int = 8, kv_heads: int = 2, history: int = 600, sequences: int = 4, nodes: int = 12,
        steps: int = 4, check: bool = False, seed: int = 0) -> float:
    """Returns the largest error of a checked output relative to the largest value (0 unchecked)."""

    device = torch.device("cuda", torch.cuda.current_device())
    g, host = torch.Generator(device=device).manual_seed(seed), torch.Generator().manual_seed(seed)

    def draw(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device=device).to(torch.bfloat16)

    frequencies, _ = rotary_frequencies(HEAD_DIM, device=device)
    reserve = steps * nodes
    width = (history + reserve) // PAGE_ROWS + 2
    pages = width + sequences * (reserve // PAGE_ROWS + 2)
    error = torch.zeros(1, dtype=torch.int32, device=device)
    pools = torch.zeros(2 * layers, kv_heads, pages * PAGE_ROWS, HEAD_DIM, dtype=torch.bfloat16, device=device)

    # the history of sequence 0, appended like a prompt
    held = -(-history // PAGE_ROWS)
    table = torch.full((1, width), -1, dtype=torch.int32, device=device)
    table[0, :held] = torch.arange(held, device=device)
    refs = torch.zeros(pages, dtype=torch.int32, device=device)
    refs[:held] = 1
    lengths = torch.zeros(1, dtype=torch.int32, device=device)
    dense = []
    for layer in range(layers):
        key, value = draw(1, history, kv_heads, HEAD_DIM), draw(1, history, kv_heads, HEAD_DIM)
        append_rows(key, value, pools[2 * layer], pools[2 * layer + 1], table, lengths, frequencies=frequencies, device_error=error)
        at = torch.arange(history, device=device)
        dense.append([[turned(key[0], at, frequencies), value[0]] for _ in range(sequences)] if check else [])
    lengths += history

    parents0 = torch.zeros(sequences, dtype=torch.int32, device=device)
    table, lengths, refs = fork_pages(pools, table, lengths, refs, parents0, reserve_rows=reserve, device_error=error)
    shared = history // PAGE_ROWS * PAGE_ROWS
    worst = 0.0
    for step in range(steps):
        parents, counts = random_trees(sequences, nodes, host)
        live = torch.tensor(counts, dtype=torch.int32, device=device)
        masks, positions = draft_tree(torch.tensor(parents, dtype=torch.int32, device=device), lengths, counts=live, device_error=error)
        scores = torch.zeros(sequences, nodes, device=device)
        drafted = []
        for layer in range(layers):
            query = draw(sequences, nodes, heads, HEAD_DIM)
            key, value = (draw(sequences, nodes, kv_heads, HEAD_DIM) for _ in range(2))
            pool = pools[2 * layer], pools[2 * layer + 1]
            q = append_rows(key, value, *pool, table, lengths, counts=live, positions=positions, frequencies=frequencies,
                            query=query, device_error=error)
            out = tree_attention(q, *pool, table, lengths, masks, HEAD_DIM ** -0.5, counts=live, shared_rows=shared,
                                 device_error=error)
            scores += out.float().square().mean(dim=(2, 3))
            drafted.append((key, value))
            for b in range(sequences if check else 0):
                same = rotate(query[b], positions[b], frequencies)
                if not torch.equal(q[b, :counts[b]], same[:counts[b]]):
                    raise RuntimeError("a query rotated by itself differs from one rotated along with an append")
                new = turned(key[b], positions[b], frequencies), value[b]
                for i in range(counts[b]):
                    path = path_to(parents[b], i)
                    k, v = (torch.cat((t, n[path])) for t, n in zip(dense[layer][b], new))
                    worst = max(worst, float((out[b, i] - dense_attention(q[b, i], k, v)).abs().max() / v.abs().max()))
        # the path to the drafted row that scores best is accepted
        scores = torch.where(torch.arange(nodes, device=device) < live[:, None], scores, -1.0)
        paths = [path_to(parents[b], int(leaf)) for b, leaf in enumerate(scores.argmax(dim=1))]
        path = torch.full((sequences, nodes), -1, dtype=torch.int32)
        for b, p in enumerate(paths):
            path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
            for layer in range(layers if check else 0):
                key, value = drafted[layer]
                rows = dense[layer][b]
                dense[layer][b] = [torch.cat((rows[0], turned(key[b], positions[b], frequencies)[p])), torch.cat((rows[1], value[b, p]))]
        lengths = keep_rows(pools, table, lengths, path.to(device), device_error=error)
        print(f"step {step}: kept {[len(p) for p in paths]} of {counts} rows, lengths {lengths.tolist()}")
    if int(error):
        raise RuntimeError(f"device error word {int(error):#x}")
    return worst


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    for name, value in (("layers", 3), ("heads", 8), ("kv-heads", 2), ("history", 600), ("sequences", 4), ("nodes", 12),
                        ("steps", 4)):
        parser.add_argument(f"--{name}", type=int, default=value)
    parser.add_argument("--check", action="store_true")
    worst = run(**vars(parser.parse_args()))
    print(f"largest error {worst:.2e} of the largest value")


if __name__ == "__main__":
    main()
