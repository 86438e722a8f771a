"""Drafted trees whose items are of every number of blocks, so that a CTA passes from one to the next at every
place of its ring of tiles, alone or with both tiles at once. Tolerances: those of ``test_drafts_gpu``."""

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


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch,nodes,heads,kv", [
    (150, 9, 8, 1),    # 72 rows: one tile a block, in turn
    (40, 20, 16, 2),   # 160 rows: both tiles
    (40, 36, 8, 1),    # 288 rows: both tiles, then one
    (30, 70, 8, 2),    # 280 rows of few heads
])
def test_items_of_every_length(batch, nodes, heads, kv, kind) -> None:
    rng = np.random.default_rng(batch)
    lengths = 128 * rng.permutation(np.arange(batch) % 9) + rng.integers(0, 130, batch)
    counts = rng.integers(nodes // 2, nodes + 1, batch)
    counts[:3] = (0, 1, nodes)
    base._attend(lengths, counts, heads, kv, nodes=nodes, kind=kind, seed=batch)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("nodes,shared", [(9, 0), (36, 0), (9, 20), (36, 33)])
def test_items_of_more_blocks_than_a_warp_has_lanes(nodes, shared, kind) -> None:
    lengths = [128 * n + d for n, d in ((31, 120), (32, -3), (33, 0), (64, 1), (70, 77))]
    base._attend(lengths, [nodes, 1, nodes, nodes - 2, nodes], 8, 1, nodes=nodes, shared=shared, kind=kind, seed=nodes)


@pytest.mark.parametrize("nodes", [9, 36])
def test_a_late_page_that_is_none(nodes) -> None:
    """Is flagged, and the next call is as if it had not been."""

    from h3sa._lib import DEVERR_BAD_PAGE
    from h3sa.drafts import tree_attention

    gen = torch.Generator().manual_seed(nodes)
    k = torch.randn(1, 90 * 128, 128, generator=gen).bfloat16().cuda()
    q = torch.randn(2, nodes, 8, 128, generator=gen).bfloat16().cuda()
    masks = base._dev(od.words(np.tri(nodes, dtype=bool)[None].repeat(2, 0)))
    good = np.stack([np.arange(45), 45 + np.arange(45)])
    lengths = base._dev([44 * 128, 43 * 128])
    want = tree_attention(q, k, k, base._dev(good), lengths, masks, base.SCALE)
    for at, page in ((40, -1), (33, 90), (0, -1)):
        bad, err = good.copy(), base._error()
        bad[1, at] = page
        tree_attention(q, k, k, base._dev(bad), lengths, masks, base.SCALE, device_error=err)
        assert int(err) & DEVERR_BAD_PAGE
        assert torch.equal(tree_attention(q, k, k, base._dev(good), lengths, masks, base.SCALE), want)
