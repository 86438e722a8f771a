"""Drafted trees over the pages of a ledger, against the oracle in 64 bits.

Tolerances, fixed before the first run. Attention, per element, from roundings of half a step (bf16 2^-8, fp16
2^-11 of the value):

    bf16:  the output 2^-8, P in bf16 2^-8, fp32 sums and the approximate 2^x 2^-12 of sum p |v|
    e4m3:  the output 2^-8, P in fp16 2^-11 and the query's two e4m3 terms, each off by 2^-17 of the row's
           maximum, so a score by scale * 2^-17 max|q| sum|k| < 2^-11 here and a weight by twice that: 2^-9
           in all of sum p |v|; weights below fp16's last step 2^-32 of the largest: 2^-30 * max p * sum |v|

The log-sum-exp is fp32: 2^-13, and 2^-11 where e4m3 scores are that far off. Bits, positions, moved rows and V of bf16 pools are exact.
Rotated keys: fp32 products and angles off by under 2^-20 of |x| + |y|, then one rounding to the pool's type,
2^-8 (bf16) or 2^-4 (e4m3, at least half of its smallest step, 2^-10) of the value.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafts as od

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _dev(a, dtype=torch.int32) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def _error() -> torch.Tensor:
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def _trees(rng, batch, nodes, roots=1):
    parents = np.full((batch, nodes), -1)
    for i in range(roots, nodes):
        parents[:, i] = rng.integers(max(0, i - 9), i, batch)
    return parents


def _table(rng, rows, shared=0, spare=3):
    """Pages of sequences with `rows` rows; the first `shared` are the same for those that have as many."""

    held = [-(-int(n) // 128) for n in rows]
    pages = shared + sum(max(0, n - shared) if n >= shared else n for n in held) + spare
    ids = rng.permutation(pages)
    table = np.full((len(held), max([1, *held])), -1, np.int64)
    at = shared
    for b, n in enumerate(held):
        mine = shared if n >= shared else 0
        table[b, :mine] = ids[:mine]
        table[b, mine:n] = ids[at:at + n - mine]
        at += n - mine
    return table, pages


def _pool(gen, kv, pages, kind):
    x = torch.randn(kv, pages * 128, 128, generator=gen)
    if kind == "bf16":
        return x.bfloat16(), None
    scale = x.abs().amax((1, 2)) / 448.0 * torch.tensor([1.0 + 0.7 * h for h in range(kv)])
    return (x / scale[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _raw(pool):
    return pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)


def _poison(pool, used):
    """NaN, infinities and the type's lowest value in every row that `used` leaves out."""

    pool = pool.clone()
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), -3.0e38])
    if pool.dtype == torch.float8_e4m3fn:
        bad = torch.tensor([float("nan"), 448.0, -448.0, float("nan")])
    rows = bad.repeat(32).to(pool.dtype)
    _raw(pool)[:, torch.from_numpy(np.flatnonzero(~used))] = _raw(rows)
    return pool


# ------------------------------------------------------------------------------------ trees


@pytest.mark.parametrize("batch,nodes", [(1, 1), (2, 9), (3, 31), (2, 32), (2, 33), (5, 128), (3, 129), (2, 500), (2, 1024)])
def test_tree_bits_and_positions(batch, nodes) -> None:
    from h3sa.drafts import draft_tree

    rng = np.random.default_rng(nodes)
    parents = _trees(rng, batch, nodes, roots=min(nodes, 2))
    parents[0] = np.arange(nodes) - 1  # a chain
    counts = rng.integers(0, nodes + 1, batch)
    counts[0] = nodes
    lengths = rng.integers(0, 1 << 20, batch)
    for given in (counts, None):
        err = _error()
        masks, positions = draft_tree(_dev(parents), _dev(lengths), counts=None if given is None else _dev(given), device_error=err)
        sees = od.ancestors(parents, np.full(batch, nodes) if given is None else given)
        assert np.array_equal(masks.cpu().numpy(), od.words(sees))
        assert np.array_equal(positions.cpu().numpy(), np.where(sees.any(-1), lengths[:, None] + sees.sum(-1) - 1, 0))
        assert int(err) == 0


def test_tree_flags_what_is_no_parent() -> None:
    from h3sa._lib import DEVERR_BAD_INDEX
    from h3sa.drafts import draft_tree

    good = np.tile(np.arange(140) - 1, (3, 1))
    for at, parent, live in ((7, 7, True), (7, 8, True), (5, -2, True), (0, 0, True), (139, 1 << 30, True), (100, 100, False)):
        parents, counts, err = good.copy(), np.array([140, 90, 140]), _error()
        parents[1 if not live else 0, at] = parent
        masks, _ = draft_tree(_dev(parents), _dev([0, 0, 0]), counts=_dev(counts), device_error=err)
        assert int(err) == (DEVERR_BAD_INDEX if live else 0)
        assert np.array_equal(masks.cpu().numpy(), od.words(od.ancestors(parents, counts)))
    for counts in ([-1, 3, 3], [3, 141, 3]):
        err = _error()
        masks, _ = draft_tree(_dev(good), _dev([0, 0, 0]), counts=_dev(counts), device_error=err)
        assert int(err) == DEVERR_BAD_INDEX
        assert np.array_equal(masks.cpu().numpy(), od.words(od.ancestors(good, np.clip(counts, 0, 140))))


def test_tree_of_nothing() -> None:
    from h3sa.drafts import draft_tree

    for shape in ((0, 5), (3, 0)):
        masks, positions = draft_tree(_dev(np.zeros(shape)), _dev(np.zeros(shape[0])))
        assert masks.shape == (*shape, 1 if shape[1] else 0) and positions.shape == shape


# ------------------------------------------------------------------------------------ append


def _append(batch, rows, heads, kv, *, kind="bf16", pairs=64, interleaved=False, axes=1, factor=1.0, positions="i32",
            seed=0, cut=True, view=lambda t: t, in_place=False, with_counts=True):
    from h3sa.drafts import append_rows
    from h3sa.rotary import rotary_frequencies

    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    counts = rng.integers(0, rows + 1, batch) if with_counts else np.full(batch, rows)
    counts[0] = rows
    lengths = rng.integers(0, 300, batch)
    table, pages = _table(rng, lengths + counts)
    (k, ks), (v, vs) = _pool(gen, kv, pages, kind), _pool(gen, kv, pages, kind)
    new_k, new_v = (torch.randn(batch, rows, kv, 128, generator=gen).bfloat16() for _ in range(2))
    if kind == "e4m3":  # some past the largest number
        new_k[:, :, :, 5], new_v[:, :, :, 9] = new_k[:, :, :, 5] * 4, new_v[:, :, :, 9] * 8
    q = torch.randn(batch, rows, heads, 128, generator=gen).bfloat16() if heads else None
    frequencies = rotary_frequencies(2 * pairs // axes, base=5e5)[0].repeat(axes, 1) if pairs else None
    where = {"i32": lambda: torch.from_numpy(rng.integers(-5000, 200000, (batch, rows, axes))).int(),
             "i64": lambda: torch.from_numpy(rng.integers(0, 1 << 40, (batch, rows, axes))),
             "f64": lambda: torch.from_numpy(rng.uniform(0, 5000, (batch, rows, axes))),
             None: lambda: torch.from_numpy(lengths[:, None, None] + np.arange(rows)[:, None])}[positions]()
    dk, dv = k.cuda(), v.cuda()
    err = _error()
    given = {} if positions is None else dict(positions=(where if axes > 1 else where[..., 0]).cuda().contiguous())
    scales = {} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda())
    dq = None if q is None else view(q.cuda())
    out = append_rows(view(new_k.cuda()), view(new_v.cuda()), dk, dv, _dev(table), _dev(lengths),
                      counts=_dev(counts) if with_counts else None,
                      frequencies=None if frequencies is None else frequencies.cuda(), interleaved=interleaved,
                      factor=factor, query=dq, query_out=dq if in_place else None, device_error=err, **given, **scales)
    torch.cuda.synchronize()
    assert int(err) == 0
    turn = lambda x: x.double() if not pairs else od.rotate(x, where, frequencies, interleaved, factor)  # noqa: E731
    want_k, want_v = turn(new_k), new_v.double()
    # Angles p f come out of 64-bit products: the oracle's is off by 2^-53 of itself, the kernel's p (f / 2 pi) by 2^-54
    # (the constant) and 2^-53 (f / 2 pi rounded; the fraction of a turn loses nothing more). Below 2^32 that
    # is under 2^-20; positions to 2^40 as here add 2^-51 |p f| to each side of a pair.
    far = 0.0 if not pairs else 2.0 ** -51 * (where.double().abs()[..., None] * frequencies).amax((-1, -2))[..., None, None]
    slack_k = (2.0 ** -20 + far) * 2 * new_k.abs().amax(-1, keepdim=True).double() * abs(factor)
    half = 2.0 ** -8 if kind == "bf16" else 2.0 ** -4
    for got, old, want, slack, scale in ((dk, k, want_k, slack_k, ks), (dv, v, want_v, 0 * slack_k, vs)):
        got, left = got.cpu(), np.ones(pages * 128, bool)
        for b in range(batch):
            at = od.places(table, b, lengths[b] + np.arange(counts[b]))
            left[at.numpy()] = False
            w = want[b, :counts[b]].transpose(0, 1)
            if scale is not None:
                w = (w / scale.double()[:, None, None]).clamp(-448, 448)
                tol = (half * w.abs()).clamp(min=2.0 ** -10) + slack[b, :counts[b]].transpose(0, 1) / scale.double()[:, None, None]
            else:
                tol = half * w.abs() + slack[b, :counts[b]].transpose(0, 1)
            assert ((got[:, at].double() - w).abs() <= tol * (1 + 1e-12)).all()
            if kind == "bf16" and want is want_v:
                assert torch.equal(got[:, at], new_v[b, :counts[b]].transpose(0, 1))
        rest = torch.from_numpy(np.flatnonzero(left))
        assert torch.equal(_raw(got)[:, rest], _raw(old)[:, rest])  # rows that nobody appended stay
    if heads:
        live = torch.arange(rows)[None] < torch.from_numpy(counts)[:, None]
        want = torch.where(live[..., None, None], turn(q), 0.0)
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -20 + far) * 2 * q.abs().amax(-1, keepdim=True).double() * abs(factor)
        assert ((out.double().cpu() - want).abs() <= tol).all()
        assert (out.cpu()[~live] == 0).all()
        assert (out.data_ptr() == dq.data_ptr()) == in_place
    else:
        assert out is None


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("batch,rows,heads,kv", [(1, 1, 1, 1), (2, 1, 3, 3), (5, 13, 8, 2), (3, 150, 0, 1), (2, 700, 4, 4), (40, 7, 14, 2)])
def test_append_sizes(batch, rows, heads, kv, kind) -> None:
    _append(batch, rows, heads, kv, kind=kind, seed=rows)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("pairs,axes,positions,kind", [
    (64, 1, None, "bf16"), (64, 1, "i64", "bf16"), (48, 3, "f64", "bf16"), (32, 1, "i32", "e4m3"), (0, 1, "i32", "bf16"),
    (36, 3, "i32", "bf16"), (12, 1, "i32", "e4m3"), (5, 1, "i32", "bf16"), (3, 3, "f64", "e4m3"), (63, 1, None, "bf16")])
def test_append_rotations(pairs, axes, positions, kind, interleaved) -> None:
    _append(4, 17, 6, 2, pairs=pairs, axes=axes, positions=positions, kind=kind, interleaved=interleaved, factor=1.2)


def test_append_strides_and_in_place() -> None:
    def merged(t):  # a slice of a merged projection
        wide = torch.full((t.shape[0], t.shape[1], 3 * t.shape[2], 128), 9.0, dtype=t.dtype, device=t.device)
        wide[:, :, t.shape[2]:2 * t.shape[2]] = t
        return wide[:, :, t.shape[2]:2 * t.shape[2]]

    def odd(t):  # rows that start at an odd element
        wide = torch.zeros(*t.shape[:3], 131, dtype=t.dtype, device=t.device)
        wide[..., 3:] = t
        return wide[..., 3:]

    for view in (merged, odd, lambda t: t.permute(2, 1, 0, 3).contiguous().permute(2, 1, 0, 3)):
        for kind in ("bf16", "e4m3"):
            _append(3, 9, 4, 2, kind=kind, view=view)
            _append(3, 9, 4, 2, kind=kind, view=view, in_place=True, interleaved=True)
    _append(3, 9, 4, 2, with_counts=False)


def test_append_flags_rows_without_a_place() -> None:
    from h3sa._lib import DEVERR_BAD_INDEX, DEVERR_BAD_PAGE
    from h3sa.drafts import append_rows

    key = torch.randn(1, 5, 2, 128, device="cuda").bfloat16()
    for length, table, count, bits, written in ((254, [[2, 1]], 5, DEVERR_BAD_INDEX, {128 + 126, 128 + 127}), (-1, [[2, 1]], 5, DEVERR_BAD_INDEX, set()),
                                         (126, [[2, -1]], 5, DEVERR_BAD_PAGE, {2 * 128 + 126, 2 * 128 + 127}),
                                         (126, [[3, 1]], 5, DEVERR_BAD_PAGE, {128, 129, 130}), (254, [[2, 1]], 2, 0, {254, 255}),
                                         ((1 << 31) - 2, [[2, 1]], 5, DEVERR_BAD_INDEX, set())):
        pools = [torch.full((2, 3 * 128, 128), 7.0, device="cuda").bfloat16() for _ in range(2)]
        err = _error()
        append_rows(key, key, *pools, _dev(table), _dev([length]), counts=_dev([count]), device_error=err)
        assert int(err) == bits
        for pool in pools:
            assert set(torch.nonzero((pool != 7.0).any(-1).any(0)).view(-1).tolist()) == written


def test_append_of_nothing() -> None:
    from h3sa.drafts import append_rows

    pool = torch.zeros(2, 128, 128, device="cuda").bfloat16()
    for batch, rows in ((0, 3), (2, 0)):
        key = torch.zeros(batch, rows, 2, 128, device="cuda").bfloat16()
        assert append_rows(key, key, pool, pool.clone(), _dev(np.zeros((batch, 1))), _dev(np.zeros(batch))) is None


def test_append_e4m3_ends_of_the_range() -> None:
    from h3sa.drafts import append_rows

    values = torch.tensor([float("inf"), -float("inf"), float("nan"), 464.0, 465.0, -500.0, 3.0e38, 2.0 ** -10, 2.0 ** -11, -0.0] + [1.0] * 118)
    key = values.bfloat16().view(1, 1, 1, 128).cuda()
    pools = [torch.zeros(1, 128, 128, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    one = torch.ones(1, device="cuda")
    append_rows(key, key, *pools, _dev([[0]]), _dev([0]), k_scale=one, v_scale=one)
    for pool in pools:
        got = pool[0, 0].float().cpu()
        assert torch.isnan(got[2]) and torch.equal(got[[0, 1, 3, 4, 5, 6]], torch.tensor([448.0, -448.0, 448.0, 448.0, -448.0, 448.0]))
        assert got[7] in (0.0, 2.0 ** -9) and (got[8:10] == 0).all() and (got[10:] == 1).all()


# ------------------------------------------------------------------------------------ attention


def _attend(lengths, counts, heads, kv, *, nodes=None, shared=0, kind="bf16", seed=0, sees=None, view=lambda t: t, q_scale=1.5):
    from h3sa.drafts import tree_attention

    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    lengths, counts = np.asarray(lengths), np.asarray(counts)
    batch, nodes = len(lengths), max(1, counts.max()) if nodes is None else nodes
    table, pages = _table(rng, lengths + counts, shared)
    (k, ks), (v, vs) = _pool(gen, kv, pages, kind), _pool(gen, kv, pages, kind)
    if sees is None:
        sees = od.ancestors(_trees(rng, batch, nodes, roots=min(2, nodes)), counts)
    elif sees == "random":
        sees = rng.random((batch, nodes, nodes)) < rng.random((batch, nodes, 1))
    q = (torch.randn(batch, nodes, heads, 128, generator=gen) * q_scale).bfloat16()
    used = np.zeros(pages * 128, bool)
    for b in range(batch):
        used[od.places(table, b, np.arange(lengths[b] + counts[b])).numpy()] = True
    k, v = _poison(k, used), _poison(v, used)
    want, want_lse, spread, peak = od.attention(q, k, v, table, lengths, counts, sees, SCALE, ks, vs)
    scales = {} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda())
    args = (view(q.cuda()), k.cuda(), v.cuda(), _dev(table), _dev(lengths), _dev(od.words(sees)), SCALE)
    err, lse = _error(), torch.full(q.shape[:3], float("nan"), device="cuda")
    out = tree_attention(*args, counts=_dev(counts), shared_rows=128 * shared, lse=lse, device_error=err, **scales)
    again = tree_attention(*args, counts=_dev(counts), shared_rows=128 * shared, **scales)
    torch.cuda.synchronize()
    assert int(err) == 0
    assert torch.equal(out, again)
    tol = (2.0 ** -7 + 2.0 ** -12) * spread if kind == "bf16" else (2.0 ** -8 + 2.0 ** -9) * spread + 2.0 ** -30 * peak
    assert torch.isfinite(out.float()).all()
    off = (out.double().cpu() - want).abs()
    assert (off <= tol).all(), float((off / tol.clamp(min=1e-30)).max())
    got = lse.double().cpu()
    assert torch.equal(got == float("-inf"), want_lse == float("-inf"))
    seen = want_lse > float("-inf")
    assert ((got - want_lse).abs()[seen] <= (2.0 ** -13 if kind == "bf16" else 2.0 ** -11)).all()


SHAPES = [
    ([0], [1], 1, 1, 0),                                  # one node, no history
    ([1, 0], [1, 0], 3, 3, 0),                            # an idle slot
    ([311, 200], [9, 4], 3, 3, 0),                        # whole items of the warp line
    ([127, 128, 129, 250], [3, 2, 1, 6], 4, 2, 0),        # nodes over page ends
    ([900, 1000, 30], [13, 1, 7], 8, 2, 0),               # the warp line's pieces
    ([700] * 6, [5, 5, 0, 3, 5, 5], 32, 4, 0),            # 40 rows
    ([513, 800, 640, 0], [9, 2, 8, 3], 8, 1, 0),          # 72 rows: the tensor line's own items
    ([1300, 95], [30, 25], 4, 1, 0),                      # 120 rows, one tile
    ([1300, 95], [60, 31], 4, 1, 0),                      # 240 rows, two tiles
    ([640, 200, 0], [150, 129, 150], 2, 2, 0),            # more nodes than a block
    ([100, 60], [300, 260], 1, 1, 0),                     # 300 rows, nodes over three blocks
    ([600, 500, 512, 100, 0], [9, 7, 3, 5, 2], 4, 2, 4),  # shared pages, sequences that end in front of them
    ([1400, 1300, 1290], [33, 20, 33], 2, 1, 10),         # shared, 198 stacked rows
    ([1500, 1700], [70, 64], 4, 1, 10),                   # joint
    ([256, 256], [1, 1], 4, 4, 2),                        # nodes right behind the shared pages
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,counts,heads,kv,shared", SHAPES)
def test_tree_attention(lengths, counts, heads, kv, shared, kind) -> None:
    _attend(lengths, counts, heads, kv, shared=shared, kind=kind)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,counts,heads,kv,shared", SHAPES)
def test_any_mask(lengths, counts, heads, kv, shared, kind) -> None:
    """Masks that are no trees, some of them empty, rows wider than any sequence's nodes, bits set behind them."""

    _attend(lengths, counts, heads, kv, shared=shared, kind=kind, sees="random", seed=1, nodes=max(counts) + 3)


def test_tree_attention_strided_query() -> None:
    def merged(q):
        wide = torch.full((q.shape[0], q.shape[1], 3 * q.shape[2], 128), 9.0, dtype=q.dtype, device=q.device)
        wide[:, :, q.shape[2]:2 * q.shape[2]] = q
        return wide[:, :, q.shape[2]:2 * q.shape[2]]

    for view in (merged, lambda q: q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)):
        _attend([300, 391], [5, 4], 6, 2, view=view)
        _attend([300, 391], [50, 44], 6, 2, view=view)


def test_a_chain_is_causal_attention() -> None:
    """The last rows of a sequence as a chain of nodes: the same result as attention to a chain."""

    from h3sa.branches import shared_prefix_attention
    from h3sa.drafts import draft_tree, tree_attention

    rng, gen = np.random.default_rng(2), torch.Generator().manual_seed(2)
    for n, heads in ((7, 4), (40, 4)):
        lengths = np.array([500, 260])
        table, pages = _table(rng, lengths + n)
        k, v = _pool(gen, 2, pages, "bf16")[0].cuda(), _pool(gen, 2, pages, "bf16")[0].cuda()
        q = torch.randn(2, n, heads, 128, generator=gen).bfloat16().cuda()
        masks, positions = draft_tree(_dev(np.tile(np.arange(n) - 1, (2, 1))), _dev(lengths))
        assert np.array_equal(positions.cpu().numpy(), lengths[:, None] + np.arange(n))
        got = tree_attention(q, k, v, _dev(table), _dev(lengths), masks, SCALE)
        want = shared_prefix_attention(q, k, v, _dev(table), _dev(lengths + n), 0, SCALE, causal=True)
        assert (got - want).abs().max() <= 2.0 ** -6 * want.abs().max()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("counts,heads,kv,length", [([6, 5], 2, 2, 200), ([20, 18], 2, 2, 1000), ([30, 31], 4, 1, 1000), ([70, 40], 4, 1, 1003), ([150, 140], 2, 2, 500)])
def test_bad_numbers_of_a_node_reach_those_that_see_it(counts, heads, kv, length, kind) -> None:
    """NaN and infinities in K and V of some nodes: rows that see none of them are as they would be without, the
    others as the formula has it."""

    from h3sa.drafts import tree_attention

    rng, gen = np.random.default_rng(5), torch.Generator().manual_seed(5)
    lengths, counts = np.array([length, length + 57]), np.array(counts)
    nodes = counts.max()
    table, pages = _table(rng, lengths + counts)
    (k, ks), (v, vs) = _pool(gen, kv, pages, kind), _pool(gen, kv, pages, kind)
    sees = od.ancestors(_trees(rng, 2, nodes, roots=3), counts)
    q = torch.randn(2, nodes, heads, 128, generator=gen).bfloat16()
    scales = {} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda())

    def run(k, v):
        return tree_attention(q.cuda(), k.cuda(), v.cuda(), _dev(table), _dev(lengths), _dev(od.words(sees)), SCALE,
                              counts=_dev(counts), **scales).float().cpu()

    clean = run(k, v)
    inf = float("nan") if kind == "e4m3" else float("inf")
    bad_k, bad_v = [0, nodes // 2], [1, nodes - 3]  # nodes
    k2, v2 = k.clone(), v.clone()
    want = clean.clone()
    for b in range(2):
        for n in bad_k:
            if n < counts[b]:
                _raw(k2)[:, od.places(table, b, [lengths[b] + n])] = _raw(torch.full((128,), float("nan")).to(k.dtype))
                want[b, sees[b, :, n]] = float("nan")
        for n, column, x in ((bad_v[0], 3, inf), (bad_v[0], 77, float("nan")), (bad_v[1], 3, -inf), (bad_v[1], 120, -inf)):
            if n < counts[b]:
                v2[:, od.places(table, b, [lengths[b] + n]), column] = torch.tensor(x).to(v.dtype)
                hit = torch.from_numpy(sees[b, :, n])
                want[b, hit, :, column] = want[b, hit, :, column] + x
    got = run(k2, v2)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))


def test_tree_attention_in_a_graph_follows_lengths_and_masks() -> None:
    from h3sa.drafts import draft_tree, tree_attention

    rng, gen = np.random.default_rng(6), torch.Generator().manual_seed(6)
    for nodes, heads in ((9, 4), (40, 4)):
        table, pages = _table(rng, [1200, 1100])
        k, v = _pool(gen, 2, pages, "bf16")[0].cuda(), _pool(gen, 2, pages, "bf16")[0].cuda()
        q = torch.randn(2, nodes, heads, 128, generator=gen).bfloat16().cuda()
        t, n, c = _dev(table), _dev([700, 600]), _dev([nodes, 3])
        parents = _dev(_trees(rng, 2, nodes))

        def step(out):
            masks, _ = draft_tree(parents, n, counts=c)
            return tree_attention(q, k, v, t, n, masks, SCALE, counts=c, out=out)

        outs = [torch.empty_like(q) for _ in range(2)]
        step(outs[0])
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        for graph, out in zip(graphs, outs):
            with torch.cuda.graph(graph):
                step(out)
        for lengths, counts in (([701, 0], [nodes, 1]), ([0, 1000], [2, nodes])):
            n.copy_(_dev(lengths))
            c.copy_(_dev(counts))
            parents.copy_(_dev(_trees(rng, 2, nodes)))
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            graphs[0].replay()
            with torch.cuda.stream(side):  # two graphs at once
                graphs[1].replay()
            torch.cuda.synchronize()
            want = step(torch.empty_like(q))
            assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_tree_attention_on_its_own_stream() -> None:
    from h3sa.drafts import tree_attention

    rng, gen = np.random.default_rng(4), torch.Generator().manual_seed(4)
    table, pages = _table(rng, [400, 500])
    k, v = _pool(gen, 2, pages, "bf16")[0].cuda(), _pool(gen, 2, pages, "bf16")[0].cuda()
    q = torch.randn(2, 5, 2, 128, generator=gen).bfloat16().cuda()
    args = (q, k, v, _dev(table), _dev([300, 400]), _dev(od.words(od.ancestors(_trees(rng, 2, 5), np.array([5, 5])))), SCALE)
    want = tree_attention(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [tree_attention(*args, stream=side) for _ in range(20)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)


def test_tree_attention_flags_lengths_counts_and_pages() -> None:
    from h3sa._lib import DEVERR_BAD_INDEX, DEVERR_BAD_PAGE
    from h3sa.drafts import tree_attention

    gen = torch.Generator().manual_seed(7)
    for nodes in (5, 90):
        k = torch.randn(2, 5 * 128, 128, generator=gen).bfloat16().cuda()
        q = torch.randn(2, nodes, 2, 128, generator=gen).bfloat16().cuda()
        masks = _dev(od.words(np.tri(nodes, dtype=bool)[None].repeat(2, 0)))
        good = [[0, 1, 2], [3, 4, 2]]
        for table, lengths, counts, bits in ((good, [100, 294], [nodes, 2], 0), (good, [-1, 100], [nodes, 2], DEVERR_BAD_INDEX),
                                             (good, [100, 385], [nodes, 0], DEVERR_BAD_INDEX), (good, [100, 383], [3, 2], DEVERR_BAD_INDEX),
                                             (good, [100, 100], [3, nodes + 1], DEVERR_BAD_INDEX), (good, [100, 100], [-1, 2], DEVERR_BAD_INDEX),
                                             ([[0, -1, 2], [3, 4, 2]], [200, 100], [1, 1], DEVERR_BAD_PAGE),
                                             ([[0, 5, 2], [3, 4, 2]], [126, 100], [3, 1], DEVERR_BAD_PAGE)):
            err = _error()
            tree_attention(q, k, k, _dev(table), _dev(lengths), masks, SCALE, counts=_dev(counts), device_error=err)
            assert int(err) == bits


def test_tree_attention_of_nothing() -> None:
    from h3sa.drafts import tree_attention

    pool = torch.zeros(1, 128, 128, device="cuda").bfloat16()
    for batch, nodes in ((0, 3), (2, 0)):
        q = torch.zeros(batch, nodes, 2, 128, device="cuda").bfloat16()
        masks = _dev(np.zeros((batch, nodes, 1 if nodes else 0)))
        assert tree_attention(q, pool, pool, _dev(np.zeros((batch, 1))), _dev(np.zeros(batch)), masks, SCALE).shape == q.shape


# ------------------------------------------------------------------------------------ keep


@pytest.mark.parametrize("batch,nodes,steps,tensors,heads,d,dtype", [
    (2, 9, 4, 2, 3, 128, torch.bfloat16), (5, 40, 12, 3, 2, 128, torch.bfloat16), (1, 200, 70, 1, 1, 128, torch.float8_e4m3fn),
    (3, 64, 64, 2, 1, 200, torch.float32), (24, 64, 8, 130, 1, 8, torch.bfloat16), (2, 9, 0, 2, 3, 128, torch.bfloat16), (2, 1, 1, 1, 1, 128, torch.bfloat16)])
def test_keep_moves_rows(batch, nodes, steps, tensors, heads, d, dtype) -> None:
    from h3sa.drafts import keep_rows

    rng, gen = np.random.default_rng(nodes), torch.Generator().manual_seed(nodes)
    lengths = rng.integers(0, 300, batch)
    table, pages = _table(rng, lengths + nodes)
    path = np.full((batch, steps), -1)
    for b in range(batch):
        n = rng.integers(0, min(nodes, steps) + 1) if b else min(nodes, steps)
        path[b, :n] = np.sort(rng.permutation(nodes)[:n])
    if steps > 2:
        path[-1, 1] = -7  # any negative ends it
    pools = torch.randn(tensors, heads, pages * 128, d, generator=gen).to(dtype)
    for stacked in (True, False):
        dev, err = pools.cuda(), _error()
        kept = keep_rows(dev if stacked else list(dev), _dev(table), _dev(lengths), _dev(path), device_error=err)
        want = od.keep(pools.view(torch.uint8).view(tensors, heads, pages * 128, -1), table, lengths, path)
        assert int(err) == 0
        assert np.array_equal(kept.cpu().numpy(), want[1])
        assert torch.equal(dev.cpu().view(torch.uint8).view(want[0].shape), want[0])


def test_keep_refuses_bad_paths_on_the_device() -> None:
    from h3sa._lib import DEVERR_BAD_INDEX, DEVERR_BAD_PAGE
    from h3sa.drafts import keep_rows

    rng = np.random.default_rng(0)
    pools = torch.from_numpy(rng.standard_normal((3, 2, 4 * 128, 128))).bfloat16()
    good = [[0, 1], [2, 3]]
    for table, lengths, path, bits in ((good, [100, 200], [[0, 2, 2], [1, 3, -1]], DEVERR_BAD_INDEX),
                                       (good, [100, 200], [[3, 2, 4], [1, 3, -1]], DEVERR_BAD_INDEX),
                                       (good, [100, 200], [[0, 2, 156], [1, 3, -1]], DEVERR_BAD_INDEX),
                                       (good, [-1, 200], [[0, 2, 3], [1, 3, -1]], DEVERR_BAD_INDEX),
                                       (good, [1 << 30, 200], [[0, 2, 1 << 30], [1, 3, -1]], DEVERR_BAD_INDEX),
                                       ([[0, -1], [2, 3]], [100, 200], [[0, 2, 40], [1, 3, -1]], DEVERR_BAD_PAGE),
                                       ([[4, 1], [2, 3]], [100, 200], [[0, 2, 40], [1, 3, -1]], DEVERR_BAD_PAGE)):
        dev, err = pools.cuda(), _error()
        kept = keep_rows(dev, _dev(table), _dev(lengths), _dev(path), device_error=err)
        assert int(err) == bits
        only = np.array(path)
        only[0] = -1  # the other sequence's path is kept
        want = od.keep(pools, np.array(table), np.array([0, 200]), only)
        assert torch.equal(dev.cpu(), want[0]) and kept.tolist() == [lengths[0], 202]


# ------------------------------------------------------------------------------------ more of each


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,counts,heads,kv,shared,nodes", [
    ([200] * 300, [1, 2, 0] * 100, 2, 1, 1, 2),                     # more sequences than are stacked by live rows
    ([400] * 90, [0, 1, 0, 2, 0, 0] * 15, 4, 2, 3, 2),              # most of them without a node
    ([700] * 9, [0] * 9, 4, 2, 5, 3),                               # none has a node
    ([1300] * 12, [30, 0, 7, 31, 1, 30, 2, 0, 0, 29, 31, 0], 4, 1, 10, 31),  # tiles that end inside sequences
    ([640, 639, 641, 0, 650], [20, 20, 1, 0, 20], 4, 1, 5, 20),     # one that ends a row in front of the shared pages' end
])
def test_stacked_rows_are_those_that_there_are(lengths, counts, heads, kv, shared, nodes, kind) -> None:
    _attend(lengths, counts, heads, kv, shared=shared, kind=kind, nodes=nodes, seed=3)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("counts,heads", [([8, 5, 8, 3], 4), ([16, 9, 1, 16], 4), ([50, 64, 3, 33], 4)])
def test_long_tables_take_the_tensor_cores(counts, heads, kind) -> None:
    """Tables wide enough that trees of more than 16 rows leave the warp line, with little in them."""

    from h3sa.drafts import tree_attention

    rng, gen = np.random.default_rng(8), torch.Generator().manual_seed(8)
    lengths, counts, nodes = np.array([300, 1000, 0, 1]), np.array(counts), max(counts)
    table, pages = _table(rng, lengths + counts)
    wide = np.full((4, 8000), -1)
    wide[:, :table.shape[1]] = table
    (k, ks), (v, vs) = _pool(gen, 2, pages, kind), _pool(gen, 2, pages, kind)
    sees = od.ancestors(_trees(rng, 4, nodes), counts)
    q = torch.randn(4, nodes, 2 * heads, 128, generator=gen).bfloat16()
    want, _, spread, peak = od.attention(q, k, v, table, lengths, counts, sees, SCALE, ks, vs)
    scales = {} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda())
    err = _error()
    out = tree_attention(q.cuda(), k.cuda(), v.cuda(), _dev(wide), _dev(lengths), _dev(od.words(sees)), SCALE, counts=_dev(counts),
                         device_error=err, **scales)
    tol = (2.0 ** -7 + 2.0 ** -12) * spread if kind == "bf16" else (2.0 ** -8 + 2.0 ** -9) * spread + 2.0 ** -30 * peak
    assert int(err) == 0 and ((out.double().cpu() - want).abs() <= tol).all()


def test_garbage_in_unused_rows_of_the_query_stays_there() -> None:
    """Queries behind the counts may hold anything."""

    from h3sa.drafts import tree_attention

    rng, gen = np.random.default_rng(9), torch.Generator().manual_seed(9)
    for nodes, shared in ((9, 0), (20, 0), (70, 0), (20, 2)):
        lengths, counts = np.array([400, 300, 0]), np.array([nodes - 3, nodes, 0])
        table, pages = _table(rng, lengths + counts, shared)
        k, v = _pool(gen, 2, pages, "bf16")[0].cuda(), _pool(gen, 2, pages, "bf16")[0].cuda()
        masks = _dev(od.words(od.ancestors(_trees(rng, 3, nodes), counts)))
        q = torch.randn(3, nodes, 4, 128, generator=gen).bfloat16().cuda()
        run = lambda q: tree_attention(q, k, v, _dev(table), _dev(lengths), masks, SCALE, counts=_dev(counts), shared_rows=128 * shared)  # noqa: E731
        want = run(q)
        for b, n in enumerate(counts):
            q[b, n:] = torch.tensor([float("nan"), float("inf"), -3.0e38, -float("inf")]).bfloat16().repeat(32).cuda()
        assert torch.equal(run(q), want)


def test_offsets_past_32_bits() -> None:
    """Pools of more than 2^31 elements: rows of the last page are appended, attended to and kept."""

    from h3sa.drafts import append_rows, keep_rows, tree_attention

    gen = torch.Generator().manual_seed(10)
    pages = 66000
    pools = torch.empty(2, 2, pages * 128, 128, dtype=torch.bfloat16, device="cuda")
    small = torch.empty(2, 2, 2 * 128, 128, dtype=torch.bfloat16, device="cuda")
    lengths, counts = _dev([120]), _dev([20])
    key, value, query = (torch.randn(1, 20, 2, 128, generator=gen).bfloat16().cuda() for _ in range(3))
    base = torch.randn(2, 2, 128, 128, generator=gen).bfloat16().cuda()
    masks = _dev(od.words(np.tri(20, dtype=bool)[None]))
    outs = []
    for p, table in ((pools, [[pages - 1, pages - 2]]), (small, [[1, 0]])):
        p[:, :, table[0][0] * 128:table[0][0] * 128 + 128] = base
        err = _error()
        append_rows(key, value, p[0], p[1], _dev(table), lengths, counts=counts, device_error=err)
        out = tree_attention(query, p[0], p[1], _dev(table), lengths, masks, SCALE, counts=counts, device_error=err)
        kept = keep_rows(p, _dev(table), lengths, _dev([[2, 7, 19]]), device_error=err)
        assert int(err) == 0 and kept.tolist() == [123]
        outs.append((out, p[:, :, table[0][0] * 128:table[0][0] * 128 + 128].clone(), p[:, :, table[0][1] * 128:table[0][1] * 128 + 12].clone()))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_appends_in_two_graphs_and_on_another_stream() -> None:
    from h3sa.drafts import append_rows, keep_rows
    from h3sa.rotary import rotary_frequencies

    gen = torch.Generator().manual_seed(11)
    f = rotary_frequencies(128)[0].cuda()
    key, query = (torch.randn(2, 7, 2, 128, generator=gen).bfloat16().cuda() for _ in range(2))
    table, lengths, counts = _dev([[0, 1], [2, 3]]), _dev([100, 124]), _dev([7, 5])
    path = _dev([[0, 3, 6], [1, -1, -1]])
    pools = [torch.zeros(2, 2, 4 * 128, 128, device="cuda").bfloat16() for _ in range(3)]
    outs = [torch.empty_like(query) for _ in range(2)]
    kept = [None, None]

    def step(p, out):
        append_rows(key, key, p[0], p[1], table, lengths, counts=counts, frequencies=f, query=query, query_out=out)
        return keep_rows(p, table, lengths, path)

    step(pools[2], outs[0])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, graph in enumerate(graphs):
        with torch.cuda.graph(graph):
            kept[i] = step(pools[i], outs[i])
    lengths.copy_(_dev([3, 125]))
    counts.copy_(_dev([7, 2]))
    for p in pools:
        p.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    out = append_rows(key, key, pools[2][0], pools[2][1], table, lengths, counts=counts, frequencies=f, query=query, stream=side)
    last = keep_rows(pools[2], table, lengths, path, stream=side)
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(pools[i], pools[2]) and torch.equal(outs[i], out) and torch.equal(kept[i], last)


def test_wrappers_refuse() -> None:
    from h3sa import drafts
    from h3sa.rotary import rotary_frequencies, rotate

    f = rotary_frequencies(128)[0].cuda()
    key = torch.zeros(2, 3, 2, 128, device="cuda").bfloat16()
    pool = torch.zeros(2, 2 * 128, 128, device="cuda").bfloat16()
    table, lengths, masks = _dev([[0], [1]]), _dev([0, 0]), _dev(np.zeros((2, 3, 1)))

    def append(match, *change, **kw):
        args = dict(key=key, value=key, key_pool=pool, value_pool=pool, table=table, lengths=lengths)
        args.update(dict(change), **kw)
        with pytest.raises(RuntimeError, match=match):
            drafts.append_rows(**args)

    append("key must be bf16", key=key.float())
    append("key must be bf16", key=key[0])
    append("value must be", value=key[:, :2])
    append("KV pools", key_pool=pool[:1])
    append("KV pools", value_pool=pool.float())
    append("bf16 or e4m3", key_pool=pool.float(), value_pool=pool.float())
    append("take no scales", k_scale=lengths.float(), v_scale=lengths.float())
    append("need k_scale", key_pool=pool.to(torch.float8_e4m3fn), value_pool=pool.to(torch.float8_e4m3fn))
    append("table", table=table[0])
    append("lengths", lengths=lengths.long())
    append("counts", counts=lengths[:1])
    append("frequencies", frequencies=f.float())
    append("do not fit", frequencies=torch.cat((f, f)))
    append("axes need positions", frequencies=f.view(2, 32))
    append("positions must be", frequencies=f, positions=lengths)
    append("positions must be contiguous", frequencies=f, positions=key[..., 0, 0].float())
    append("query must be", query=key[:, :2])
    append("query_out", query=key, query_out=key[:, :2])
    append("without a query", query_out=key)
    append("rows of key", key=key.transpose(2, 3).contiguous().transpose(2, 3))
    append("int32 tensor", device_error=lengths.long())
    append("require CUDA", key=key.cpu())
    query = torch.zeros(2, 3, 4, 128, device="cuda").bfloat16()
    for match, change in (("masks", dict(masks=masks[:, :, 0])), ("masks", dict(masks=masks.long())), ("query", dict(query=query[0])),
                          ("counts", dict(counts=lengths[:1])), ("shared rows", dict(shared_rows=256)), ("shared rows", dict(shared_rows=64)),
                          ("scale", dict(softmax_scale=0.0)), ("require CUDA", dict(query=query.cpu(), masks=masks.cpu()))):
        args = dict(query=query, key_pool=pool, value_pool=pool, table=table, lengths=lengths, masks=masks, softmax_scale=0.1)
        args.update(change)
        with pytest.raises(RuntimeError, match=match):
            drafts.tree_attention(**args)
    for match, args in (("parents", (lengths, lengths)), ("parents", (masks[..., 0].long(), lengths)), ("lengths", (masks[..., 0], lengths[:1])),
                        ("at most 1024", (_dev(np.zeros((1, 1025))), lengths[:1])), ("require CUDA", (masks[..., 0].cpu(), lengths.cpu()))):
        with pytest.raises(RuntimeError, match=match):
            drafts.draft_tree(*args)
    for match, args in (("pool tensors", ([pool[0]], table, lengths, masks[..., 0])), ("no pool tensors", ([], table, lengths, masks[..., 0])),
                        ("pool tensors", ([pool[:, :100]], table, lengths, masks[..., 0])), ("path", ([pool], table, lengths, lengths)),
                        ("path", ([pool], table, lengths, masks[:1, :, 0])), ("lengths", ([pool], table, lengths.long(), masks[..., 0])),
                        ("row bytes", (torch.zeros(1, 1, 128, 3, device="cuda"), table, lengths, masks[..., 0].contiguous()))):
        with pytest.raises(RuntimeError, match=match):
            drafts.keep_rows(*args)
    x, at = torch.zeros(5, 2, 128, device="cuda"), torch.zeros(5, dtype=torch.int32, device="cuda")
    for match, args, kw in (("bf16, fp16 or fp32", (x.double(), at, f), {}), ("bf16, fp16 or fp32", (x[0], at, f), {}),
                            ("positions", (x, at[:4], f), {}), ("positions", (x, at.float(), f), {}), ("do not fit", (x[..., :64], at, f), {}),
                            ("positions", (x, at, f.view(2, 32)), {}), ("float64", (x, at, f.float()), {}), ("out must be", (x, at, f), dict(out=x.half())),
                            ("contiguous", (x.transpose(1, 2).contiguous().transpose(1, 2), at, f), {}), ("finite", (x, at, f), dict(factor=float("inf"))),
                            ("at most 1024", (torch.zeros(5, 1, 1026, device="cuda"), at, f), {}), ("require CUDA", (x.cpu(), at, f), {})):
        with pytest.raises(RuntimeError, match=match):
            rotate(*args, **kw)
