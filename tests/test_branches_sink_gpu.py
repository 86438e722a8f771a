"""Attention over a sink: one key that takes nearly all weight, with a value of zero, in front of or
behind thousands of equal keys far below it, whose values make up the whole output. What a format of P
loses at small weights shows here in full, as every key of the tail is rounded the same way.

Tolerance, fixed before the first run, relative to the output (all values are positive, so the output
is sum p |v|): 2^-8 for the rounding of the output to bf16; of a weight, 2^-8 for P in bf16, and for e4m3
pools, whose P has 11 bits down to 2^-21 of the largest weight and steps of 2^-31 of it below, 2^-10
down to weights of 2^-22; fp32 sums of 15000 terms, 16 and more at a time, 2^-13; scores of 22 log2
units in fp32, 2^-18. Together (2^-7 + 2^-9) for bf16 and (2^-8 + 2^-9) for e4m3.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import branches as ob

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _exact(value, v_scale, lengths, table, group, sink, depth):
    """fp64 output and log-sum-exp of a row, [batch, heads, 128] and [batch]: one weight of 1 with a
    value of zero and a tail of weights 2^-depth; tail scores are 0."""

    outs, lses = [], []
    for b, n in enumerate(lengths):
        at = torch.tensor([int(table[b, j // 128]) * 128 + j % 128 for j in range(n) if j != sink[b]], device="cuda")
        total = 1.0 + (n - 1) * 2.0 ** -depth[b]
        mean = value[:, at].double().sum(1) * (2.0 ** -depth[b] / total)
        if v_scale is not None:
            mean = mean * v_scale.double()[:, None]
        outs.append(mean.repeat_interleave(group, 0))
        lses.append(depth[b] * math.log(2.0) + math.log(total))
    return torch.stack(outs), torch.tensor(lses, dtype=torch.float64, device="cuda")


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,shared,rows,heads,kv", [
    ([3000, 2800], 0, 130, 64, 64),                      # both tiles, items that a CTA has nearly whole
    ([2900, 3100, 2700], 0, 20, 96, 24),                 # 80 rows an item: one tile
    ([40100 + 3 * b for b in range(20)], 313, 1, 8, 8),  # 20 stacked rows over shared keys: four copies
    ([20500 + 3 * b for b in range(30)], 160, 1, 16, 8), # 60: two copies
    ([15000], 0, 600, 24, 24),                           # long items of two tiles
    ([1500 + b for b in range(150)], 0, 1, 8, 8),        # few rows, a whole item a warp
    ([500 + b for b in range(40)], 0, 2, 8, 8),          # short tables
])
@pytest.mark.parametrize("depth", [15.3, 17.6, 19.27, 21.8])
@pytest.mark.parametrize("late", [False, True])
def test_tail_behind_a_sink(lengths, shared, rows, heads, kv, kind, depth, late) -> None:
    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(17)
    gen = torch.Generator(device="cuda").manual_seed(17)
    width = max(ob.pages_of(n) for n in lengths)
    pages = shared + sum(ob.pages_of(n) - shared for n in lengths) + 1
    ids, at = rng.permutation(pages), shared
    table = np.full((len(lengths), width), -1, np.int64)
    for b, n in enumerate(lengths):
        table[b, :shared] = ids[:shared]
        table[b, shared:ob.pages_of(n)] = ids[at:at + ob.pages_of(n) - shared]
        at += ob.pages_of(n) - shared
    # the sink: the first key of all, or one in the middle
    where = [(min(lengths) if shared == 0 else shared * 128) // 2 + 5 if late else 0 for _ in lengths]
    value = torch.rand(kv, pages * 128, 128, generator=gen, device="cuda") + 0.5
    key = torch.zeros_like(value)
    for b in range(len(lengths)):
        row = int(table[b, where[b] // 128]) * 128 + where[b] % 128
        key[:, row] = 1.0
        value[:, row] = 0.0
    # a query of ones times the sink's ones: 128 * unit * (k_scale) * SCALE * log2 e is the depth
    want_unit = depth / (128 * SCALE * math.log2(math.e))
    if kind == "bf16":
        q_value = torch.tensor(want_unit).bfloat16()
        key, value, scales = key.bfloat16(), value.bfloat16(), {}
        real = float(q_value) * 128 * SCALE * math.log2(math.e)
        v_scale = None
    else:
        k_scale = torch.full((kv,), want_unit / 448, dtype=torch.float32, device="cuda")
        v_scale = torch.full((kv,), 1.5 / 448, dtype=torch.float32, device="cuda")
        q_value = torch.tensor(1.0)
        key = (key * 448).to(torch.float8_e4m3fn)
        value = (value * (448 / 1.5)).to(torch.float8_e4m3fn)
        scales = dict(k_scale=k_scale, v_scale=v_scale)
        real = float(k_scale[0].double()) * 448 * 128 * SCALE * math.log2(math.e)
    q = torch.full((len(lengths), rows, heads, 128), float(q_value), dtype=torch.bfloat16, device="cuda")
    lse = torch.empty(q.shape[:3], device="cuda")
    out = shared_prefix_attention(q, key, value, torch.from_numpy(table).to(torch.int32).cuda(),
                                  torch.tensor(lengths, dtype=torch.int32, device="cuda"), shared * 128, SCALE,
                                  lse=lse, **scales)
    want, want_lse = _exact(value, v_scale, lengths, table, heads // kv, where, [real] * len(lengths))
    tol = 2.0 ** -7 + 2.0 ** -9 if kind == "bf16" else 2.0 ** -8 + 2.0 ** -9
    off = (out.double() / want[:, None] - 1).abs()
    assert off.max() <= tol, float(off.max())
    assert ((lse.double() - want_lse[:, None, None]).abs() <= 2.0 ** -13).all()
