"""Paths of the branch operators that sizes alone reach: more pool tensors than one copy launch takes, a
captured graph of both attention lines and the merge, tiles of few stacked rows against shared keys on the
tensor cores. The ledger is exact; attention is held against an uncaptured call bit for bit, or against
fp64 within the bounds of test_branches_gpu.py.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import branches as ob

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _i32(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()


@pytest.mark.parametrize("count", [127, 128, 129, 257])
@pytest.mark.parametrize("listed", [False, True])
def test_many_pool_tensors(count, listed) -> None:
    from h3sa.branches import compact_pages, fork_pages

    rng = np.random.default_rng(count)
    pages, width = 24, 6
    table = np.full((3, width), -1, np.int64)
    ids = rng.permutation(pages)
    table[0, :3], table[1, :2], table[2, :4] = ids[:3], ids[3:5], ids[5:9]
    lengths, refs = np.array([300, 256, 511]), np.bincount(table[table >= 0], minlength=pages)
    pools = torch.from_numpy(rng.integers(0, 1 << 15, (count, 2, pages * 128, 8))).to(torch.int16)
    give = lambda t: list(t.unbind(0)) if listed else t  # noqa: E731
    dev = pools.cuda()
    parents = np.array([2, 0, -1, 2])
    *want, moves = ob.fork(table, lengths, refs, parents, reserve_rows=130)
    got = fork_pages(give(dev), _i32(table), _i32(lengths), _i32(refs), _i32(parents), reserve_rows=130)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    pools = ob.copy_rows(pools, moves)
    assert torch.equal(dev.cpu(), pools)
    want_table, want_refs, live, moves = ob.compact(table, refs)
    assert moves
    got = compact_pages(give(dev), _i32(table), _i32(refs))
    for g, w in zip(got, (want_table, want_refs, [live])):
        np.testing.assert_array_equal(g.cpu().numpy(), w)
    assert torch.equal(dev.cpu(), ob.copy_rows(pools, moves))


def _ragged(lengths, shared, rng):
    width = max([shared] + [ob.pages_of(n) for n in lengths])
    pages = shared + sum(max(0, ob.pages_of(n) - shared) for n in lengths) + 1
    ids, at = rng.permutation(pages), shared
    table = np.full((len(lengths), width), -1, np.int64)
    for b, n in enumerate(lengths):
        held = ob.pages_of(n)
        table[b, :shared] = ids[:shared]
        table[b, shared:held] = ids[at:at + held - shared]
        at += held - shared
    return table, pages


def _pools(kv, pages, kind, gen):
    k, v = (torch.randn(kv, pages * 128, 128, generator=gen, device="cuda") for _ in range(2))
    if kind == "bf16":
        return k.bfloat16(), v.bfloat16(), {}
    k, v = ((t * 64).clamp(-448, 448).to(torch.float8_e4m3fn) for t in (k, v))
    scale = lambda: (1.0 + torch.arange(kv, device="cuda") / 8) / 64  # noqa: E731
    return k, v, dict(k_scale=scale(), v_scale=scale())


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch,shared,rows,heads,kv", [
    (24, 64, 4, 32, 8),    # shared keys on the tensor cores, own ones on the warp line, and the merge
    (6, 4, 100, 6, 6),     # joint
    (3, 9, 70, 2, 2),      # all on the tensor cores, split
])
def test_graph_of_both_lines(batch, shared, rows, heads, kv, kind) -> None:
    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(7)
    gen = torch.Generator(device="cuda").manual_seed(7)
    most = shared * 128 + 900
    table, pages = _ragged([most] * batch, shared, rng)
    k, v, scales = _pools(kv, pages, kind, gen)
    q = torch.randn(batch, rows, heads, 128, generator=gen, device="cuda").bfloat16()
    t, n = _i32(table), _i32([most] * batch)
    out, lse = torch.empty_like(q), torch.empty(batch, rows, heads, device="cuda")
    call = lambda o, s: shared_prefix_attention(q, k, v, t, n, shared * 128, SCALE, causal=True, out=o, lse=s, **scales)  # noqa: E731
    call(out, lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, lse)
    for low in (0, 40, shared * 128, shared * 128 + 1):
        lengths = rng.integers(low, most + 1, batch)
        lengths[rng.integers(batch)] = most
        n.copy_(_i32(lengths))
        out.fill_(7.0)
        graph.replay()
        lse2 = torch.empty_like(lse)
        assert torch.equal(out, call(None, lse2)) and torch.equal(lse, lse2)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,shared,rows,heads,kv", [
    ([40100 + 40 * b for b in range(20)], 313, 1, 8, 8),   # 20 stacked rows: four copies
    ([20500 + 37 * b for b in range(15)], 160, 1, 32, 8),  # 60: two copies
    ([26000 + 11 * b for b in range(11)], 203, 3, 8, 8),   # 33
    ([200, 20500, 20400, 0, 20485] + [20480] * 12, 160, 1, 32, 8),  # some shorter than the prefix
])
@pytest.mark.parametrize("causal", [False, True])
def test_few_stacked_rows_on_the_tensor_cores(lengths, shared, rows, heads, kv, kind, causal) -> None:
    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(13)
    gen = torch.Generator(device="cuda").manual_seed(13)
    table, pages = _ragged([max(n, shared * 128) for n in lengths], shared, rng)
    k, v, scales = _pools(kv, pages, kind, gen)
    q = (torch.randn(len(lengths), rows, heads, 128, generator=gen, device="cuda") * 1.5).bfloat16()
    lse = torch.empty(q.shape[:3], device="cuda")
    out = shared_prefix_attention(q, k, v, _i32(table), _i32(lengths), shared * 128, SCALE, causal=causal, lse=lse, **scales)
    group = heads // kv
    for b, n in enumerate(lengths):
        if n == 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        at = torch.from_numpy(table[b, np.arange(n) // 128] * 128 + np.arange(n) % 128).cuda()
        for h in range(kv):
            raw = [p[h].view(torch.uint8 if kind == "e4m3" else torch.int16)[at].view(p.dtype).double() for p in (k, v)]
            key, value = raw if kind == "bf16" else (raw[0] * scales["k_scale"][h].double(), raw[1] * scales["v_scale"][h].double())
            x = q[b, :, h * group:(h + 1) * group].double() @ key.T * SCALE
            if causal:
                limit = n - (rows - 1) + torch.arange(rows, device="cuda")
                x.masked_fill_((torch.arange(n, device="cuda") >= limit[:, None])[:, None], -math.inf)
            w = torch.softmax(x, -1)
            want, spread = w @ value, w @ value.abs()
            peak = w.amax(-1, keepdim=True) * ((x > -math.inf).double() @ value.abs())
            tol = ((2.0 ** -7 + 2.0 ** -12) * spread if kind == "bf16" else
                   (2.0 ** -7 + 2.0 ** -11) * spread + 2.0 ** -15 * peak)
            got = out[b, :, h * group:(h + 1) * group].double()
            assert ((got - want).abs() <= tol).all()
            assert ((lse[b, :, h * group:(h + 1) * group].double() - torch.logsumexp(x, -1)).abs() <= 2.0 ** -13).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rows,heads,kv", [(1, 4, 2), (70, 2, 2), (300, 40, 40)])
def test_visible_infinities_of_v_reach_their_column_alone(rows, heads, kv, kind) -> None:
    """As infinities or, where a form multiplies them with zeros of P, as NaN."""

    from h3sa.branches import shared_prefix_attention

    gen = torch.Generator(device="cuda").manual_seed(19)
    k, v, scales = _pools(kv, 5, kind, gen)
    q = torch.randn(2, rows, heads, 128, generator=gen, device="cuda").bfloat16()
    args = (_i32([[2, 0, 1], [2, 3, 4]]), _i32([300, 384]), 128, SCALE)
    want = shared_prefix_attention(q, k, v, *args, **scales)
    bad = float("inf") if kind == "bf16" else float("nan")
    raw = v.view(torch.uint8) if kind == "e4m3" else v
    raw[0, 3 * 128 + 77, 11] = 0x7f if kind == "e4m3" else bad  # a row of sequence 1 alone
    out = shared_prefix_attention(q, k, v, *args, **scales)
    hit = out[1, :, :heads // kv, 11].float()
    assert not torch.isfinite(hit).any()
    out[1, :, :heads // kv, 11] = want[1, :, :heads // kv, 11]
    assert torch.equal(out, want)
