"""Infinities and NaN in V of drafted rows where several warps, tiles or CTAs share their item's blocks.

All comparisons are exact: other rows and columns are what they are without the bad values, and what sees one is infinite
or NaN."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import numpy as np
import pytest
import torch

from oracle import drafts as od

_spec = importlib.util.spec_from_file_location("drafts_gpu", Path(__file__).with_name("test_drafts_gpu.py"))
base = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(base)

pytestmark = pytest.mark.gpu


class _Call:
    """A call of tree_attention whose pools can be changed between runs."""

    def __init__(self, lengths, counts, heads, kv, sees, *, kind="bf16", seed=0):
        rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
        self.lengths, self.counts, self.kind = np.array(lengths), np.array(counts), kind
        self.table, pages = base._table(rng, self.lengths + self.counts)
        (self.k, ks), (self.v, vs) = base._pool(gen, kv, pages, kind), base._pool(gen, kv, pages, kind)
        self.q = torch.randn(len(lengths), max(counts), heads, 128, generator=gen).bfloat16()
        self.scales = {} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda())
        self.sees = sees
        self.args = base._dev(self.table), base._dev(self.lengths), base._dev(od.words(sees))

    def node(self, b, n):
        return od.places(self.table, b, [self.lengths[b] + n])

    def __call__(self, k, v, times=1):
        args = self.q.cuda(), k.cuda(), v.cuda(), *self.args, base.SCALE
        from h3sa.drafts import tree_attention

        outs = [tree_attention(*args, counts=base._dev(self.counts), **self.scales) for _ in range(times)]
        assert all(torch.equal(o.view(torch.int16), outs[0].view(torch.int16)) for o in outs[1:])
        return outs[0].float().cpu()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("seen_by", [0, 40])  # a row of the item's first tile, one of its second
def test_values_that_one_tile_alone_sees(seen_by, kind) -> None:
    """Items of 200 rows: both MMA warps clear each block, the rows of one tile alone see the node."""

    lengths, counts = [128 * (i % 5) + 37 * (i % 7) for i in range(40)], [50] * 40
    sees = np.zeros((40, 50, 50), bool)
    sees[:, np.arange(50), np.arange(50)] = True
    call = _Call(lengths, counts, 16, 4, sees, kind=kind)
    want = call(call.k, call.v)
    v = call.v.clone()
    for b in range(40):
        for column, x in ((5, float("nan")), (127, float("nan") if kind == "e4m3" else float("inf"))):
            v[:, call.node(b, seen_by), column] = torch.tensor(x).to(v.dtype)
            want[b, seen_by, :, column] = x
    got = call(call.k, v, times=50)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


@pytest.mark.parametrize("nodes", [24, 48])  # 96 rows: one tile; 192: both
def test_an_infinity_stays_in_its_item(nodes) -> None:
    """CTAs go on from an item whose node holds an infinity to the first blocks of the next, all of whose weight is in
    later blocks: nodes score far above the history, whose part in the output vanishes. What the node adds is infinite and
    not infinity times a vanished weight."""

    lengths, counts = [1100 + 13 * i for i in range(24)], [nodes] * 24
    sees = np.tri(nodes, dtype=bool)[None].repeat(24, 0)
    call = _Call(lengths, counts, 32, 8, sees)
    call.q = torch.full_like(call.q, 1.5)
    k, v = call.k.clone(), call.v.clone()
    for b in range(24):
        for n in range(nodes):
            k[:, call.node(b, n)] = 40.0
        v[:, call.node(b, 0), 7] = float("inf")
    want = call(k, call.v)
    want[..., 7] = float("inf")
    assert torch.equal(call(k, v), want)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,nodes,heads,kv", [([128 * 30 + 100] * 2, 60, 8, 1), ([128 * 70 + 127, 900, 20], 24, 4, 1), ([700, 40], 9, 4, 2)])
def test_nodes_of_several_blocks_and_pieces(lengths, nodes, heads, kv, kind) -> None:
    """Bad values in nodes on both sides of a page's end, seen by some rows each."""

    counts = [nodes - i for i in range(len(lengths))]
    rng = np.random.default_rng(3)
    sees = rng.random((len(lengths), nodes, nodes)) < 0.3
    sees &= (np.arange(nodes) < np.array(counts)[:, None])[:, None, :]
    call = _Call(lengths, counts, heads, kv, sees, kind=kind)
    want, v = call(call.k, call.v), call.v.clone()
    for b, count in enumerate(counts):
        for n, column in ((0, 3), (count // 2, 64), (count - 1, 127), (count - 1, 3)):
            v[:, call.node(b, n), column] = torch.tensor(float("nan")).to(v.dtype)
            want[b, :count, :, column][torch.from_numpy(sees[b, :count, n])] = float("nan")
    got = call(call.k, v, times=3)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
