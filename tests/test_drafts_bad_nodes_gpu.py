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
