"""Attention over a shared prefix and the page ledger around it, against the CPU oracle.

Tolerances, fixed before the first run. Attention: the score products are exact and summed in
fp32, so weights are off by rounding only: bf16 P by at most 2^-8 of each weight (8 significant
bits, round to nearest), the two e4m3 terms of P by at most 2^-8 of it (4 + 4 significant bits)
and by 2^-16 of the largest weight where the second term reaches e4m3's smallest step; the output
is rounded once to bf16 (2^-8). Everything else (fp32 sums, the approximate 2^x, the e4m3 terms of
the query) stays below 2^-12 of a weight. An element may therefore be off by

    bf16:  (2^-8 + 2^-8 + 2^-12) * sum p |v|
    e4m3:  (2^-8 + 2^-8 + 2^-11) * sum p |v| + 2^-15 * max p * sum |v|

The log-sum-exp is fp32 throughout: 2^-13 absolute covers sums of some thousand terms. The ledger
operations and the row copies are exact.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import branches as ob

pytestmark = pytest.mark.gpu
SCALE = 128 ** -0.5


def _i32(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).cuda()


def _batch(lengths, shared, rng, spare=3):
    """Table of sequences that share `shared` pages and hold scattered pages of their own; entries
    past a sequence's end are -1."""

    width = max([shared] + [ob.pages_of(n) for n in lengths] + [1])
    pages = shared + sum(max(0, ob.pages_of(n) - shared) for n in lengths) + spare
    ids = rng.permutation(pages)
    table = np.full((len(lengths), width), -1, np.int64)
    at = shared
    for b, n in enumerate(lengths):
        held = ob.pages_of(n)
        table[b, :min(held, shared)] = ids[:min(held, shared)]
        for j in range(shared, held):
            table[b, j] = ids[at]
            at += 1
    return table, pages


def _pool(gen, kv, pages, kind):
    x = torch.randn(kv, pages * 128, 128, generator=gen)
    if kind == "bf16":
        return x.bfloat16(), None
    scale = x.abs().amax((1, 2)) / 448.0 * torch.tensor([1.0 + 0.7 * h for h in range(kv)])
    return (x / scale[:, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _poison(pool, table, lengths, shared):
    """NaN, infinities and the type's lowest value in every row that no sequence has."""

    used = np.zeros(pool.shape[1], bool)
    for b, n in enumerate(lengths):
        for j in range(n):
            used[table[b, j // 128] * 128 + j % 128] = True
    pool = pool.clone()
    idle = torch.from_numpy(np.flatnonzero(~used))
    bad = torch.tensor([float("nan"), float("inf"), -float("inf"), -3.0e38])
    if pool.dtype == torch.float8_e4m3fn:
        bad = torch.tensor([float("nan"), 448.0, -448.0, float("nan")])
    rows = bad.repeat(32).to(pool.dtype)
    raw = pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)
    raw[:, idle] = rows.view(raw.dtype)
    return pool


def _check(lengths, shared, rows, heads, kv, kind="bf16", causal=False, seed=0, q_scale=1.5,
           query=None, poison=True):
    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    lengths = np.asarray(lengths)
    table, pages = _batch(lengths, shared, rng)
    (k, ks), (v, vs) = _pool(gen, kv, pages, kind), _pool(gen, kv, pages, kind)
    q = (torch.randn(len(lengths), rows, heads, 128, generator=gen) * q_scale).bfloat16()
    if poison:
        k, v = _poison(k, table, lengths, shared), _poison(v, table, lengths, shared)
    want, want_lse, spread, peak = ob.attention(q, k, v, table, lengths, SCALE, causal=causal,
                                                k_scale=ks, v_scale=vs)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse = torch.full(q.shape[:3], float("nan"), device="cuda")
    scales = {} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda())
    dq = q.cuda() if query is None else query(q.cuda())
    args = (dq, k.cuda(), v.cuda(), _i32(table), _i32(lengths), shared * 128, SCALE)
    out = shared_prefix_attention(*args, causal=causal, lse=lse, device_error=err, **scales)
    again = shared_prefix_attention(*args, causal=causal, **scales)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert torch.equal(out, again)
    if kind == "bf16":
        tol = (2.0 ** -7 + 2.0 ** -12) * spread
    else:
        tol = (2.0 ** -7 + 2.0 ** -11) * spread + 2.0 ** -15 * peak
    off = (out.double().cpu() - want).abs()
    assert torch.isfinite(out.float()).all()
    assert (off <= tol).all(), float((off / tol.clamp(min=1e-30)).max())
    got = lse.double().cpu()
    assert torch.equal(got == float("-inf"), want_lse == float("-inf"))
    seen = want_lse > float("-inf")
    assert ((got - want_lse).abs()[seen] <= 2.0 ** -13).all()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("lengths,shared,rows,heads,kv", [
    ([1], 0, 1, 1, 1),                                    # one key
    ([256, 257], 2, 1, 3, 3),                             # a branch with no row of its own
    ([300, 0, 384, 513, 1, 130], 1, 1, 14, 2),            # an idle slot, one shorter than the prefix
    ([127, 128, 129], 0, 2, 4, 2),                        # nothing shared
    ([700] * 40, 4, 1, 4, 4),                             # 40 stacked rows: two copies
    ([520, 777, 641], 4, 33, 2, 1),                       # 198 stacked rows: two tiles
    ([1500, 1700, 1536], 10, 7, 8, 1),                    # 168 rows, 56 own rows an item
    ([400, 650], 2, 150, 2, 1),                           # own items of two tiles
    ([900, 300], 2, 600, 1, 1),                           # joint, with a last tile of 88 rows
    ([640, 200, 0], 1, 515, 2, 2),                        # joint, an idle sequence
    ([0, 0], 1, 3, 2, 2),                                 # nobody sees anything
])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_matches_oracle(lengths, shared, rows, heads, kv, kind, causal) -> None:
    _check(lengths, shared, rows, heads, kv, kind, causal)


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_attention_sharp_and_rising_scores(kind) -> None:
    """Large scores: the running maximum keeps growing along the sequence, so O is rescaled often
    and late keys take nearly all weight."""

    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(3)
    gen = torch.Generator().manual_seed(3)
    lengths = np.array([1290, 1400])
    table, pages = _batch(lengths, 8, rng)
    (k, ks), (v, vs) = _pool(gen, 1, pages, kind), _pool(gen, 1, pages, kind)
    if kind == "bf16":
        k = (k.float() * 0.2).bfloat16()
    order = torch.zeros(pages * 128)
    for b in range(2):
        for j in range(int(lengths[b])):
            order[table[b, j // 128] * 128 + j % 128] = j / 1400
    ramp = order[None, :, None] * (12.0 if kind == "bf16" else 150.0)
    k = (k.float() + ramp).clamp(-448, 448).to(k.dtype)
    q = (torch.randn(2, 3, 2, 128, generator=gen) * 0.3 + 0.25).bfloat16()
    want, want_lse, spread, peak = ob.attention(q, k, v, table, lengths, SCALE, k_scale=ks, v_scale=vs)
    scales = {} if ks is None else dict(k_scale=ks.cuda(), v_scale=vs.cuda())
    lse = torch.empty(2, 3, 2, device="cuda")
    out = shared_prefix_attention(q.cuda(), k.cuda(), v.cuda(), _i32(table), _i32(lengths), 1024,
                                  SCALE, lse=lse, **scales)
    tol = ((2.0 ** -7 + 2.0 ** -12) * spread if kind == "bf16" else
           (2.0 ** -7 + 2.0 ** -11) * spread + 2.0 ** -15 * peak)
    # scores of some tens: fp32 keeps them to 2^-16, which moves a weight by as much
    assert ((out.double().cpu() - want).abs() <= tol + 2.0 ** -13 * spread).all()
    assert ((lse.double().cpu() - want_lse).abs() <= 2.0 ** -11).all()


def test_attention_strided_query() -> None:
    """Queries as slices of a merged projection and transposed storage."""

    def merged(q):
        wide = torch.full((q.shape[0], q.shape[1], 3 * q.shape[2], 128), 9.0, dtype=q.dtype, device=q.device)
        wide[:, :, q.shape[2]:2 * q.shape[2]] = q
        return wide[:, :, q.shape[2]:2 * q.shape[2]]

    def heads_first(q):
        return q.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)

    for view in (merged, heads_first):
        _check([300, 391], 2, 5, 6, 2, query=view)


def test_attention_on_its_own_stream() -> None:
    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(4)
    gen = torch.Generator().manual_seed(4)
    lengths = np.array([300, 400])
    table, pages = _batch(lengths, 2, rng)
    k, v = _pool(gen, 2, pages, "bf16")[0].cuda(), _pool(gen, 2, pages, "bf16")[0].cuda()
    q = torch.randn(2, 1, 2, 128, generator=gen).bfloat16().cuda()
    t, n = _i32(table), _i32(lengths)
    want = shared_prefix_attention(q, k, v, t, n, 256, SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [shared_prefix_attention(q, k, v, t, n, 256, SCALE, stream=side) for _ in range(20)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(o, want) for o in outs)


def test_attention_in_a_graph_follows_the_lengths() -> None:
    """A captured call reads lengths and table on the device, so replays follow them."""

    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(5)
    gen = torch.Generator().manual_seed(5)
    table, pages = _batch([900, 1000], 2, rng)
    k, v = _pool(gen, 2, pages, "bf16")[0].cuda(), _pool(gen, 2, pages, "bf16")[0].cuda()
    q = torch.randn(2, 1, 4, 128, generator=gen).bfloat16().cuda()
    t, n = _i32(table), _i32([300, 270])
    out = torch.empty_like(q)
    shared_prefix_attention(q, k, v, t, n, 256, SCALE, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        shared_prefix_attention(q, k, v, t, n, 256, SCALE, out=out)
    for lengths in ([301, 271], [900, 513], [0, 1000]):
        n.copy_(_i32(lengths))
        graph.replay()
        got = out.clone()
        assert torch.equal(got, shared_prefix_attention(q, k, v, t, n, 256, SCALE))


def test_attention_pool_past_32_bits() -> None:
    """Pages whose byte and element offsets pass 2^32 and 2^31."""

    from h3sa.branches import shared_prefix_attention

    pages = 140000  # 4.6 GB a pool
    k = torch.zeros(1, pages * 128, 128, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    gen = torch.Generator().manual_seed(6)
    table = np.array([[139998, 139999, 139990], [139998, 139999, 131100]])
    small = {p: i for i, p in enumerate(sorted(set(table.reshape(-1))))}
    ks, vs = (_pool(gen, 1, len(small), "bf16")[0] for _ in range(2))
    for p, i in small.items():
        k[:, p * 128:(p + 1) * 128] = ks[:, i * 128:(i + 1) * 128].cuda()
        v[:, p * 128:(p + 1) * 128] = vs[:, i * 128:(i + 1) * 128].cuda()
    near = np.vectorize(small.get)(table)
    q = torch.randn(2, 1, 2, 128, generator=gen).bfloat16()
    lengths = np.array([300, 384])
    want, _, spread, _ = ob.attention(q, ks, vs, near, lengths, SCALE)
    out = shared_prefix_attention(q.cuda(), k, v, _i32(table), _i32(lengths), 256, SCALE)
    assert ((out.double().cpu() - want).abs() <= (2.0 ** -7 + 2.0 ** -12) * spread).all()


def test_attention_propagates_visible_nan_only_to_its_rows() -> None:
    from h3sa.branches import shared_prefix_attention

    rng = np.random.default_rng(7)
    gen = torch.Generator().manual_seed(7)
    lengths = np.array([300, 400])
    table, pages = _batch(lengths, 2, rng)
    k, v = _pool(gen, 1, pages, "bf16")[0], _pool(gen, 1, pages, "bf16")[0]
    k[0, table[1, 3] * 128 + 5] = float("nan")  # a key of sequence 1 alone
    q = torch.randn(2, 1, 2, 128, generator=gen).bfloat16()
    out = shared_prefix_attention(q.cuda(), k.cuda(), v.cuda(), _i32(table), _i32(lengths), 256, SCALE)
    assert torch.isfinite(out[0].float()).all() and torch.isnan(out[1].float()).all()


def test_attention_device_errors() -> None:
    from h3sa import _lib
    from h3sa.branches import shared_prefix_attention

    k = torch.zeros(1, 4 * 128, 128, dtype=torch.bfloat16, device="cuda")
    q = torch.zeros(1, 1, 1, 128, dtype=torch.bfloat16, device="cuda")
    for table, length, bit in (([[0, 9]], 200, _lib.DEVERR_BAD_PAGE), ([[0, -1]], 200, _lib.DEVERR_BAD_PAGE),
                               ([[0, 1]], 257, _lib.DEVERR_BAD_INDEX), ([[0, 1]], -1, _lib.DEVERR_BAD_INDEX)):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        shared_prefix_attention(q, k, k, _i32(table), _i32([length]), 0, SCALE, device_error=err)
        assert int(err.item()) == bit


# ------------------------------------------------------------------------------ the ledger


def _ledger(rng, sequences, width, pages, fill=0.6):
    table = np.full((sequences, width), -1, np.int64)
    lengths = np.zeros(sequences, np.int64)
    ids = rng.permutation(pages)
    at, room = 0, int(pages * fill)
    common: list[int] = []
    for s in range(sequences):
        if s % 3 == 0:
            n = min(int(rng.integers(0, width // 2 + 1)), room - at)
            common = list(ids[at:at + n])
            at += n
        n = min(int(rng.integers(0, width - len(common) + 1)), room - at)
        held = common + list(ids[at:at + n])
        at += n
        table[s, :len(held)] = held
        if held:
            lengths[s] = 128 * (len(held) - 1) + (int(rng.integers(1, 129)) if n else 128)
    return table, lengths, np.bincount(table[table >= 0], minlength=pages)


def _equal(got, want):
    for g, w in zip(got, want):
        assert g.dtype == torch.int32
        np.testing.assert_array_equal(g.cpu().numpy(), w)


@pytest.mark.parametrize("sequences,width,pages,children,reserve,private", [
    (1, 1, 2, 1, 0, False),
    (4, 12, 64, 2, 1, False),
    (9, 7, 200, 30, 129, False),
    (5, 9, 300, 11, 0, True),
    (3, 20, 3000, 2100, 1, False),  # more children than threads
])
@pytest.mark.parametrize("listed", [False, True])
def test_fork_matches_oracle(sequences, width, pages, children, reserve, private, listed) -> None:
    from h3sa.branches import fork_pages

    rng = np.random.default_rng(sequences * 100 + children)
    table, lengths, refs = _ledger(rng, sequences, width, pages, 0.25)
    table = np.pad(table, ((0, 0), (0, 2 + ob.pages_of(reserve))), constant_values=-1)
    parents = rng.integers(-1, sequences, children)
    parents[:min(2, children)] = 0
    *want, moves = ob.fork(table, lengths, refs, parents, reserve_rows=reserve, private=private)
    pools = torch.randn(6, 2, pages * 128, 16, generator=torch.Generator().manual_seed(1)).bfloat16()
    dev = pools.cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    given = [_i32(a) for a in (table, lengths, refs)]
    got = fork_pages(list(dev.unbind(0)) if listed else dev, *given, _i32(parents), reserve_rows=reserve,
                     private=private, device_error=err)
    assert int(err.item()) == 0
    _equal(got, want)
    _equal(given, (table, lengths, refs))  # as they were
    assert torch.equal(dev.cpu(), ob.copy_rows(pools, moves))


def test_fork_failures_leave_everything_as_it_was() -> None:
    from h3sa import _lib
    from h3sa.branches import fork_pages

    table, lengths = np.array([[2, 0, -1], [1, -1, -1]]), np.array([200, 128])
    refs = np.array([1, 1, 1, 0])
    pools = torch.randn(2, 1, 4 * 128, 8, device="cuda").bfloat16()
    before = pools.clone()

    def fails(bit, parents, reserve=0, table=table, lengths=lengths, refs=refs):
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = fork_pages(pools, _i32(table), _i32(lengths), _i32(refs), _i32(parents), reserve_rows=reserve,
                         device_error=err)
        assert int(err.item()) == bit
        _equal(got, (np.full((len(parents), 3), -1), np.zeros(len(parents)), refs))
        assert torch.equal(pools, before)

    fails(_lib.DEVERR_NO_PAGES, [0, 0])          # two partial pages, one free
    fails(_lib.DEVERR_NO_PAGES, [-1], 129)
    fails(_lib.DEVERR_BAD_INDEX, [0, 2])         # no such sequence
    fails(_lib.DEVERR_BAD_INDEX, [0], 400)       # does not fit the table row
    fails(_lib.DEVERR_BAD_INDEX, [0], lengths=np.array([-5, 128]))
    fails(_lib.DEVERR_BAD_PAGE, [0], table=np.array([[2, 7, -1], [1, -1, -1]]))
    fails(_lib.DEVERR_BAD_PAGE, [0], table=np.array([[2, 3, -1], [1, -1, -1]]))  # a free page


@pytest.mark.parametrize("sequences,width,pages", [(1, 1, 1), (5, 16, 96), (24, 40, 700), (3, 900, 5000)])
def test_compact_matches_oracle(sequences, width, pages) -> None:
    from h3sa.branches import compact_pages

    rng = np.random.default_rng(pages)
    table, _, refs = _ledger(rng, sequences, width, pages, 0.55)
    want_table, want_refs, live, moves = ob.compact(table, refs)
    pools = torch.randn(4, 1, pages * 128, 8, generator=torch.Generator().manual_seed(2)).bfloat16()
    dev = pools.cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = compact_pages(dev, _i32(table), _i32(refs), device_error=err)
    assert int(err.item()) == 0
    _equal(got, (want_table, want_refs, np.array([live])))
    assert torch.equal(dev.cpu(), ob.copy_rows(pools, moves))


def test_compact_flags_entries_of_free_pages() -> None:
    from h3sa import _lib
    from h3sa.branches import compact_pages

    pools = torch.zeros(1, 1, 4 * 128, 8, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = compact_pages(pools, _i32([[3, 1], [9, -1]]), _i32([0, 0, 0, 1]), device_error=err)
    assert int(err.item()) == _lib.DEVERR_BAD_PAGE
    _equal(got, (np.array([[0, -1], [-1, -1]]), np.array([1, 0, 0, 0]), np.array([1])))


@pytest.mark.parametrize("sequences,width,pages", [(1, 1, 1), (8, 64, 512), (256, 100, 9000)])
def test_free_matches_oracle(sequences, width, pages) -> None:
    from h3sa.branches import free_pages

    rng = np.random.default_rng(width)
    table, lengths, refs = _ledger(rng, sequences, width, pages, 1.0)
    release = rng.random(sequences) < 0.5
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = free_pages(_i32(table), _i32(lengths), _i32(refs), torch.from_numpy(release).cuda(), device_error=err)
    assert int(err.item()) == 0
    _equal(got, ob.free(table, lengths, refs, release))


def test_free_flags_references_that_are_not_there() -> None:
    from h3sa import _lib
    from h3sa.branches import free_pages

    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = free_pages(_i32([[0, 1], [5, -1]]), _i32([200, 7]), _i32([2, 0]),
                     torch.tensor([True, True], device="cuda"), device_error=err)
    assert int(err.item()) == _lib.DEVERR_BAD_PAGE
    _equal(got, (np.full((2, 2), -1), np.zeros(2), np.array([1, 0])))


def test_refusals() -> None:
    from h3sa.branches import compact_pages, fork_pages, free_pages, shared_prefix_attention

    z = lambda *shape, dtype=torch.int32: torch.zeros(*shape, dtype=dtype, device="cuda")  # noqa: E731
    k = z(2, 256, 128, dtype=torch.bfloat16)
    q = z(1, 1, 4, 128, dtype=torch.bfloat16)
    ok = dict(query=q, key_pool=k, value_pool=k, table=z(1, 2), lengths=z(1), shared_rows=0, softmax_scale=1.0)
    for change, match in (
        (dict(query=q.cpu()), "CUDA"),
        (dict(query=q.float()), "query must be bf16"),
        (dict(query=z(1, 1, 3, 128, dtype=torch.bfloat16)), "no multiple"),
        (dict(query=z(1, 1, 4, 129, dtype=torch.bfloat16)[..., 1:]), "16-byte aligned"),
        (dict(value_pool=k[:, :128].contiguous()), "KV pools"),
        (dict(key_pool=k.float(), value_pool=k.float()), "bf16 or e4m3"),
        (dict(k_scale=z(2, dtype=torch.float32)), "no scales"),
        (dict(key_pool=k.to(torch.float8_e4m3fn), value_pool=k.to(torch.float8_e4m3fn)), "need k_scale"),
        (dict(table=z(2, 2)), "table"),
        (dict(lengths=z(1, dtype=torch.int64)), "lengths"),
        (dict(shared_rows=100), "whole pages"),
        (dict(shared_rows=384), "whole pages"),
        (dict(softmax_scale=0.0), "scale"),
        (dict(softmax_scale=float("nan")), "scale"),
        (dict(out=z(1, 1, 4, 64, dtype=torch.bfloat16)), "out"),
        (dict(lse=z(1, 1, 4)), "lse"),
        (dict(device_error=z(1, dtype=torch.int64)), "device_error"),
    ):
        with pytest.raises(RuntimeError, match=match):
            shared_prefix_attention(**{**ok, **change})
    pools = z(1, 1, 256, 8, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="reference counts"):
        fork_pages(pools, z(1, 2), z(1), z(3), z(1))
    with pytest.raises(RuntimeError, match="parents"):
        fork_pages(pools, z(1, 2), z(1), z(2), z(1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="one shape and dtype"):
        fork_pages([pools[0], pools[0].bfloat16()], z(1, 2), z(1), z(2), z(1))
    with pytest.raises(ValueError, match="reserve_rows"):
        fork_pages(pools, z(1, 2), z(1), z(2), z(1), reserve_rows=-1)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        compact_pages(z(1, 1, 256, 3, dtype=torch.float32), z(1, 2), z(2))
    with pytest.raises(RuntimeError, match="release"):
        free_pages(z(1, 2), z(1), z(2), z(1))
    with pytest.raises(RuntimeError, match="table"):
        free_pages(z(1, 4)[:, ::2], z(1), z(2), z(1, dtype=torch.bool))
