"""NaN and infinities where a row does not look: queries of rows that see nothing."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import branches as ob

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _i32(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()


def _pools(kv, pages, kind, gen):
    k, v = (torch.randn(kv, pages * 128, 128, generator=gen, device="cuda") for _ in range(2))
    if kind == "bf16":
        return k.bfloat16(), v.bfloat16(), {}
    one = torch.full((kv,), 1.0 / 64, device="cuda")
    k, v = ((t * 64).clamp(-448, 448).to(torch.float8_e4m3fn) for t in (k, v))
    return k, v, dict(k_scale=one, v_scale=one)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows,heads,kv", [(100, 2, 2), (200, 2, 1), (300, 40, 40), (20, 2, 1)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_rows_that_see_nothing_whatever_their_query(rows, heads, kv, kind, bad) -> None:
    """Causal rows in front of a sequence's first key; their queries must not matter, nor touch others."""

    from h3sa.branches import shared_prefix_attention

    gen = torch.Generator(device="cuda").manual_seed(31)
    k, v, scales = _pools(kv, 3, kind, gen)
    q = torch.randn(1, rows, heads, 128, generator=gen, device="cuda").bfloat16()
    seen = rows // 2 + 3
    args = (k, v, _i32([[2, 0, 1]]), _i32([seen]), 0, SCALE)
    want = shared_prefix_attention(q, *args, causal=True, **scales)
    q[:, :rows - seen, :, 7] = bad
    lse = torch.empty(1, rows, heads, device="cuda")
    out = shared_prefix_attention(q, *args, causal=True, lse=lse, **scales)
    assert (out[:, :rows - seen] == 0).all() and (lse[:, :rows - seen] == float("-inf")).all()
    assert torch.equal(out, want) and torch.isfinite(lse[:, rows - seen:]).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows,heads,kv", [(100, 2, 2), (200, 2, 1), (300, 40, 40), (20, 2, 1)])
def test_a_query_that_is_nan_reaches_its_own_row_only(rows, heads, kv, kind) -> None:
    from h3sa.branches import shared_prefix_attention

    gen = torch.Generator(device="cuda").manual_seed(37)
    k, v, scales = _pools(kv, 6, kind, gen)
    q = torch.randn(2, rows, heads, 128, generator=gen, device="cuda").bfloat16()
    args = (k, v, _i32([[2, 0, 1], [3, 5, -1]]), _i32([300, 240]), 0, SCALE)
    want = shared_prefix_attention(q, *args, **scales)
    q[1, rows // 3, heads - 1, 9] = float("nan")
    lse = torch.empty(2, rows, heads, device="cuda")
    out = shared_prefix_attention(q, *args, lse=lse, **scales)
    assert torch.isnan(out[1, rows // 3, heads - 1]).all() and torch.isnan(lse[1, rows // 3, heads - 1])
    out[1, rows // 3, heads - 1] = want[1, rows // 3, heads - 1]
    assert torch.equal(out, want) and int(torch.isnan(lse).sum()) == 1
