"""Attention over a shared prefix at the sizes that send its work to the tensor cores' line, and at
every form of a tile there, against fp64 on the device; the small sizes are in
test_branches_gpu.py, whose bounds on the error hold here as they are: the fp32 sums grow to tens of
thousands of terms, whose roundings add up to about sqrt(terms) * 2^-24, still below 2^-12.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import branches as ob

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _dense(pool, table, n, head):
    """fp64 rows [n, 128] of one head of a sequence."""

    pages = pool[head].view(-1, 128, 128)
    held = table[: ob.pages_of(n)].long()
    return pages[held].reshape(-1, 128)[:n].double()


def _attention(q, k, v, table, lengths, causal, ks, vs):
    """(out, lse, sum p |v|, max p * sum |v|) in fp64."""

    batch, rows, heads, _ = q.shape
    kv = k.shape[0]
    group = heads // kv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    spread, peak = torch.zeros_like(out), torch.zeros_like(out)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        for h in range(kv):
            key, value = _dense(k, table[b], n, h), _dense(v, table[b], n, h)
            if ks is not None:
                key, value = key * ks[h].double(), value * vs[h].double()
            x = q[b, :, h * group:(h + 1) * group].double() @ key.T * SCALE
            if causal:
                limit = n - (rows - 1) + torch.arange(rows, device=q.device)
                x.masked_fill_((torch.arange(n, device=q.device) >= limit[:, None])[:, None], -math.inf)
            at = (b, slice(None), slice(h * group, (h + 1) * group))
            lse[at] = torch.logsumexp(x, -1)
            w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
            out[at], spread[at] = w @ value, w @ value.abs()
            peak[at] = w.amax(-1, keepdim=True) * ((x > -math.inf).double() @ value.abs())
    return out, lse, spread, peak


def _inputs(lengths, shared, rows, heads, kv, kind, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    width = max([shared] + [ob.pages_of(n) for n in lengths])
    pages = shared + sum(max(0, ob.pages_of(n) - shared) for n in lengths) + 2
    ids = rng.permutation(pages)
    table, at = np.full((len(lengths), width), -1, np.int64), shared
    for b, n in enumerate(lengths):
        held = ob.pages_of(n)
        table[b, :min(held, shared)] = ids[:min(held, shared)]
        more = max(0, held - shared)
        table[b, shared:shared + more] = ids[at:at + more]
        at += more
    pools, scales = [], []
    for _ in range(2):
        x = torch.randn(kv, pages * 128, 128, generator=gen, device="cuda")
        if kind == "bf16":
            pools.append(x.bfloat16())
            scales.append(None)
        else:
            scale = x.abs().amax((1, 2)) / 448.0 * (1.0 + 0.3 * torch.arange(kv, device="cuda"))
            pools.append((x / scale[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn))
            scales.append(scale)
    q = (torch.randn(len(lengths), rows, heads, 128, generator=gen, device="cuda") * 1.5).bfloat16()
    return q, *pools, torch.from_numpy(table).to(torch.int32).cuda(), *scales


def _check(lengths, shared, rows, heads, kv, kind, causal):
    from h3sa.branches import shared_prefix_attention

    q, k, v, table, ks, vs = _inputs(lengths, shared, rows, heads, kv, kind, seed=11)
    want, want_lse, spread, peak = _attention(q, k, v, table, lengths, causal, ks, vs)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full(q.shape[:3], float("nan"), device="cuda")
    scales = {} if ks is None else dict(k_scale=ks, v_scale=vs)
    args = (q, k, v, table, n, shared * 128, SCALE)
    out = shared_prefix_attention(*args, causal=causal, lse=lse, device_error=err, **scales)
    again = shared_prefix_attention(*args, causal=causal, **scales)
    assert int(err) == 0
    assert torch.equal(out, again)
    tol = ((2.0 ** -7 + 2.0 ** -12) * spread if kind == "bf16" else
           (2.0 ** -7 + 2.0 ** -11) * spread + 2.0 ** -15 * peak)
    off = (out.double() - want).abs()
    assert torch.isfinite(out.float()).all()
    assert (off <= tol).all(), float((off / tol.clamp(min=1e-30)).max())
    assert torch.equal(lse == -math.inf, want_lse == -math.inf)
    seen = want_lse > -math.inf
    assert ((lse.double() - want_lse).abs()[seen] <= 2.0 ** -13).all()


def test_oracles_agree() -> None:
    lengths, shared, rows, heads, kv = [300, 0, 390], 1, 3, 4, 2
    q, k, v, table, ks, vs = _inputs(lengths, shared, rows, heads, kv, "e4m3", seed=5)
    got = _attention(q, k, v, table, lengths, True, ks, vs)
    want = ob.attention(q.cpu(), k.cpu(), v.cpu(), table.cpu().numpy(), np.asarray(lengths), SCALE, causal=True,
                        k_scale=ks.cpu(), v_scale=vs.cpu())
    for a, b in zip(got, want):
        torch.testing.assert_close(a.cpu(), b, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,shared,rows,heads,kv", [
    ([31700 + 40 * b for b in range(20)], 247, 1, 8, 8),       # 20 stacked rows: four copies
    ([16500 + 37 * b for b in range(15)], 128, 1, 32, 8),      # 60: two copies
    ([16000, 17000, 16400, 16384], 128, 3, 64, 8),             # 96: one tile, unpaired
    ([8200 + 111 * b for b in range(12)], 64, 2, 64, 8),       # 192: both tiles
    ([8300 + 50 * b for b in range(13)], 64, 3, 24, 3),        # 312: a span, then four copies of 56 rows
    ([16384 + 9 * b for b in range(34)], 128, 1, 40, 8),       # 170, some with few rows of their own
    ([100, 20000, 0, 16385] + [16400] * 6, 128, 1, 64, 8),     # 80 rows, some shorter than the prefix
    ([900, 1300], 2, 70, 2, 2),                                # a branch's own: one tile
    ([900, 1300, 77], 3, 61, 8, 4),                            # 122
    ([900, 1300], 2, 100, 4, 2),                               # 200: both tiles
    ([1000, 1400], 2, 75, 8, 2),                               # 300: a span, then two copies of 44
    ([2000, 1400], 2, 69, 8, 2),                               # 276: a span, then four copies of 20
    ([5000, 3000], 3, 512, 3, 3),                              # few items of many rows
    ([2100, 2600], 3, 900, 2, 1),                              # the same, ragged
    ([1000 + 64 * b for b in range(9)], 2, 130, 8, 8),         # joint: a tile and two rows
    ([2100, 0, 2600, 700], 3, 515, 8, 8),                      # joint: two spans and three rows; an idle one
    ([900, 1300, 641, 5000], 5, 300, 16, 8),                   # joint: the last span has 88 rows
    ([700, 1300], 1, 257, 24, 24),                             # joint: one row in the last span
    ([900 + 40 * b for b in range(11)], 4, 100, 6, 6),         # joint: a tile each, not full
    ([700 + 90 * b for b in range(8)], 0, 33, 24, 8),          # the same with nothing shared, three heads a KV head
    ([3000, 2000, 1000], 7, 250, 6, 6),                        # joint, no more items than the stacked rows make
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_of_many_rows(lengths, shared, rows, heads, kv, kind, causal) -> None:
    _check(lengths, shared, rows, heads, kv, kind, causal)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,shared,rows,heads,kv", [
    ([200000], 1562, 1, 4, 1),                 # one long sequence in many parts
    ([40000, 65], 0, 1, 2, 2),                 # nothing shared: lengths far apart
    ([130] * 300, 1, 1, 8, 8),                 # many branches of two rows
    ([5000 + 64 * b for b in range(5)], 39, 2, 64, 2),    # four 16-row tiles a branch
    ([4000 + b for b in range(33)], 31, 1, 16, 16),       # lengths one apart, a tile of one row
    ([2048 + 31 * b for b in range(9)], 16, 3, 15, 3),    # own rows end inside a tile
])
def test_attention_of_few_rows(lengths, shared, rows, heads, kv, kind) -> None:
    _check(lengths, shared, rows, heads, kv, kind, False)
