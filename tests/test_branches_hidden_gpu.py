"""NaN and infinities where a row does not look: queries of rows that see nothing, and values of shared
pages behind the end of a sequence that is shorter than the prefix."""

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


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,shared,rows,heads,kv", [
    ([100, 1000, 130, 0], 6, 1, 4, 2),             # few rows
    ([300, 2000], 12, 1, 4, 4),
    ([500, 1100, 513, 0], 5, 100, 4, 2),           # tensor cores, both lines' items
    ([9000, 200] + [16500] * 8, 128, 1, 64, 8),    # shared keys on the tensor cores, own ones not
    ([900, 100], 6, 300, 40, 40),                  # joint
    ([200, 100], 4, 3, 2, 2),                      # all of them shorter than the prefix
])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_rows_of_shared_pages_behind_a_short_sequence(lengths, shared, rows, heads, kv, kind, causal, bad) -> None:
    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(41)
    gen = torch.Generator(device="cuda").manual_seed(41)
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
    k, v, scales = _pools(kv, pages, kind, gen)
    q = torch.randn(len(lengths), rows, heads, 128, generator=gen, device="cuda").bfloat16()
    args = (_i32(table), _i32(lengths), shared * 128, SCALE)
    want = shared_prefix_attention(q, k, v, *args, causal=causal, **scales)
    short = [b for b, n in enumerate(lengths) if n < shared * 128]
    first = max(lengths[b] for b in short)  # the first row that no short sequence has
    rows_of = np.concatenate([np.arange(max(first, j * 128), (j + 1) * 128) - j * 128 + ids[j] * 128
                              for j in range(first // 128, shared)])
    hidden = torch.from_numpy(rows_of).cuda()
    if kind == "bf16":
        v[:, hidden] = bad
    else:
        v.view(torch.uint8)[:, hidden] = 0x7f  # NaN, the only one of the two that e4m3 has
    out = shared_prefix_attention(q, k, v, *args, causal=causal, **scales)
    for b in short:
        assert torch.equal(out[b], want[b])
