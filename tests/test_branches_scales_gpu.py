"""e4m3 pools whose score factor is tiny or zero: query rows of zeros (padding), a head of zero keys with
the quantisers' smallest scale, a scale of zero. All visible scores are then equal (or nearly), the
output is the mean of the visible values, and hidden keys stay hidden. Tolerances as in
test_branches_gpu.py, without the term of the largest weight: all weights are alike.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import branches as ob

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _inputs(lengths, shared, rows, heads, kv, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    width = max([shared] + [ob.pages_of(n) for n in lengths])
    pages = shared + sum(max(0, ob.pages_of(n) - shared) for n in lengths) + 1
    ids, at = rng.permutation(pages), shared
    table = np.full((len(lengths), width), -1, np.int64)
    for b, n in enumerate(lengths):
        held = ob.pages_of(n)
        table[b, :min(held, shared)] = ids[:min(held, shared)]
        for j in range(shared, held):
            table[b, j] = ids[at]
            at += 1
    k, v = (torch.randn(kv, pages * 128, 128, generator=gen).mul(60).clamp(-448, 448).to(torch.float8_e4m3fn)
            for _ in range(2))
    q = torch.randn(len(lengths), rows, heads, 128, generator=gen).bfloat16()
    return table, k, v, q


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,shared,rows,heads,kv", [
    ([57, 300], 0, 1, 4, 4),             # short tables
    ([1000, 1111, 1290], 7, 2, 8, 4),    # few rows
    ([300, 333], 1, 150, 4, 4),          # both tiles
    ([390, 259], 1, 70, 4, 4),           # one tile
    ([700, 531], 2, 300, 40, 40),        # joint
])
@pytest.mark.parametrize("what", ["zero query", "smallest scale", "both", "scale of zero"])
def test_score_factor_of_nothing(lengths, shared, rows, heads, kv, what, causal) -> None:
    from h3sa.branches import shared_prefix_attention

    table, k, v, q = _inputs(lengths, shared, rows, heads, kv, seed=23)
    k_scale, v_scale = torch.full((kv,), 0.01), torch.linspace(0.01, 0.03, kv)
    if what in ("zero query", "both"):
        q[:, ::2] = 0.0
    if what in ("smallest scale", "both"):
        k[1], k_scale[1] = torch.zeros_like(k[1].float()).to(k.dtype), 1e-12
        k_scale[0] = 1e-12
    if what == "scale of zero":
        k_scale[0] = 0.0
    lse = torch.empty(q.shape[:3], device="cuda")
    i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()  # noqa: E731
    out = shared_prefix_attention(q.cuda(), k.cuda(), v.cuda(), i32(table), i32(np.asarray(lengths)), shared * 128, SCALE,
                                  causal=causal, k_scale=k_scale.cuda(), v_scale=v_scale.cuda(), lse=lse)
    few = slice(0, 2)  # the heads in question, and one beside them
    want, want_lse, spread, peak = ob.attention(q[:, :, few], k[few], v[few], table, np.asarray(lengths), SCALE,
                                                causal=causal, k_scale=k_scale[few], v_scale=v_scale[few]) \
        if heads == kv else ob.attention(q, k, v, table, np.asarray(lengths), SCALE, causal=causal, k_scale=k_scale,
                                         v_scale=v_scale)
    got, got_lse = out.double().cpu(), lse.double().cpu()
    if heads == kv:
        got, got_lse = got[:, :, few], got_lse[:, :, few]
    tol = (2.0 ** -7 + 2.0 ** -11) * spread + 2.0 ** -15 * peak
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all()
    assert torch.equal(got_lse == float("-inf"), want_lse == float("-inf"))
    seen = want_lse > float("-inf")
    assert ((got_lse - want_lse).abs()[seen] <= 2.0 ** -13).all()
