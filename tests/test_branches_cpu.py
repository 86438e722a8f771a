"""The ledger's rules on the oracle, and what the C entry points and wrappers refuse before any launch."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import branches as ob

PAGES, WIDTH = 64, 8


def _counts(table: np.ndarray) -> np.ndarray:
    return np.bincount(table[table >= 0], minlength=PAGES)


def _rows(pool: torch.Tensor, table: np.ndarray, n: int) -> torch.Tensor:
    return torch.cat([pool[:0]] + [pool[table[j] * 128:table[j] * 128 + min(128, n - 128 * j)]
                                   for j in range(ob.pages_of(n))])


@pytest.mark.parametrize("seed", range(4))
def test_ledger_keeps_rows_and_counts(seed: int) -> None:
    """Fork, free and compact in turn: every sequence keeps its rows, every count its references."""

    rng = np.random.default_rng(seed)
    pool = torch.from_numpy(rng.integers(0, 1 << 30, (PAGES * 128, 1)))
    lengths = np.array([300, 128, 0])
    table = np.full((3, WIDTH), -1)
    free = rng.permutation(PAGES)
    table[0, :3], table[1, :1] = free[:3], free[3:4]
    refs = _counts(table)
    rows = [_rows(pool, table[s], int(lengths[s])) for s in range(3)]
    for _ in range(6):
        parents = rng.integers(-1, len(lengths), 3)
        child, child_lengths, refs, moves = ob.fork(table, lengths, refs, parents, reserve_rows=int(rng.integers(0, 200)),
                                                    private=bool(rng.integers(0, 2)))
        pool = ob.copy_rows(pool, moves)
        assert len({dst for _, dst, _ in moves}) == len(moves)
        table, lengths = np.concatenate([table, child]), np.concatenate([lengths, child_lengths])
        rows += [rows[p] if p >= 0 else pool[:0] for p in parents]
        assert np.array_equal(refs, _counts(table))
        # a page behind the shared whole ones belongs to one sequence alone
        for c in range(len(lengths) - 3, len(lengths)):
            own = table[c, int(lengths[c]) // 128:]
            assert (refs[own[own >= 0]] == 1).all()
        release = rng.random(len(lengths)) < 0.4
        table, lengths, refs = ob.free(table, lengths, refs, release)
        rows = [r[:0] if gone else r for r, gone in zip(rows, release)]
        assert np.array_equal(refs, _counts(table))
        table, refs, live, moves = ob.compact(table, refs)
        pool = ob.copy_rows(pool, moves)
        assert np.array_equal(refs, _counts(table)) and (refs[:live] > 0).all() and (refs[live:] == 0).all()
        for s in range(len(lengths)):
            assert torch.equal(_rows(pool, table[s], int(lengths[s])), rows[s])


def test_attention_oracle_is_attention() -> None:
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 5 * 128, 128, generator=gen, dtype=torch.float64) for _ in range(2))
    table, lengths = np.array([[4, 1, -1], [4, 0, 2]]), np.array([200, 259])
    q = torch.randn(2, 3, 4, 128, generator=gen, dtype=torch.float64)
    out, lse, _, _ = ob.attention(q, k, v, table, lengths, 0.1, causal=True)
    for b in range(2):
        n = int(lengths[b])
        kk, vv = (torch.stack([_rows(t[h], table[b], n) for h in range(2)]).repeat_interleave(2, 0) for t in (k, v))
        hidden = torch.arange(n)[None] > torch.arange(n - 3, n)[:, None]
        x = (q[b].transpose(0, 1) @ kk.transpose(1, 2) * 0.1).masked_fill(hidden, float("-inf"))
        torch.testing.assert_close(out[b], (x.softmax(-1) @ vv).transpose(0, 1), rtol=1e-12, atol=1e-12)
        torch.testing.assert_close(lse[b], x.logsumexp(-1).T, rtol=1e-12, atol=1e-12)


P = 1 << 20  # a 16-byte aligned address that nothing dereferences


def _attend(**change) -> tuple[int, str]:
    from h3sa import _lib

    a = dict(q=P, sb=512, sn=512, sh=128, out=P, lse=None, batch=2, rows=1, heads=4, kv=2, k=P, v=P, pages=4,
             e4m3=0, ks=None, vs=None, table=P, width=4, lengths=P, shared=128, causal=0, scale=0.1, work=P,
             bytes=1 << 40, err=None, stream=None)
    a.update(change)
    return _lib.LIB.h3sa_shared_prefix_attention(*a.values()), _lib.last_error()


@pytest.mark.parametrize("change,match", [
    (dict(heads=3), "multiple of kv_heads"),
    (dict(kv=0), "invalid sizes"),
    (dict(batch=-1), "invalid sizes"),
    (dict(rows=-1), "invalid sizes"),
    (dict(pages=0), "invalid pool"),
    (dict(pages=1 << 24), "invalid pool"),
    (dict(width=0), "invalid pool"),
    (dict(width=1 << 24), "invalid pool"),
    (dict(shared=-128), "whole pages"),
    (dict(shared=64), "whole pages"),
    (dict(shared=5 * 128), "whole pages"),
    (dict(q=None), "null pointer"),
    (dict(work=None), "null pointer"),
    (dict(e4m3=1, ks=P), "null pointer"),
    (dict(scale=0.0), "scale"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(scale=float("nan")), "scale"),
    (dict(q=P + 8), "16-byte aligned"),
    (dict(k=P + 8), "16-byte aligned"),
    (dict(out=P + 4), "16-byte aligned"),
    (dict(sn=516), "16-byte aligned"),
    (dict(batch=1 << 20, rows=1 << 10, heads=4, kv=2), "too large"),
    (dict(batch=1 << 16, rows=64, width=1 << 16, pages=1 << 16), "work index"),
    (dict(bytes=64), "workspace of 64 bytes"),
])
def test_attention_entry_refuses(change, match) -> None:
    code, message = _attend(**change)
    assert code != 0 and match in message, message


def test_attention_of_nothing_is_nothing() -> None:
    assert _attend(batch=0)[0] == 0
    assert _attend(rows=0)[0] == 0


def test_workspaces_grow_with_the_work() -> None:
    from h3sa import _lib

    size = _lib.LIB.h3sa_shared_prefix_workspace
    assert size(0, 1, 1, 1, 0) == 0 and size(1, 1, 3, 2, 0) == 0 and size(1, 1, 1, 1, -1) == 0
    assert 0 < size(1, 1, 8, 8, 0) < size(64, 1, 8, 8, 0) < size(64, 1, 64, 8, 128 * 128)
    pages = _lib.LIB.h3sa_pages_workspace
    assert pages(0, 1) == 0 and pages(1, -1) == 0 and 0 < pages(10, 0) < pages(10, 8) < pages(20, 8)


def test_ledger_entries_refuse() -> None:
    from h3sa import _lib

    pools = _lib.Pools()
    pools.base, pools.stride, pools.count, pools.heads, pools.pages, pools.row_bytes = P, 4096, 1, 1, 8, 32
    fork = [P, 2, 4, P, P, P, 2, 0, 0, P, P, P, P, None, None]
    compact = [P, 2, 4, P, P, P, P, P, None, None]
    free = [P, 2, 4, P, P, 8, P, P, P, P, None, None]

    def refused(fn, *args) -> str:
        assert getattr(_lib.LIB, fn)(*args) != 0
        return _lib.last_error()

    def changed(args, **at):
        return [at.get(f"a{i}", a) for i, a in enumerate(args)]

    for at, match in ((dict(a1=-1), "invalid sizes"), (dict(a2=0), "invalid sizes"), (dict(a2=1 << 25), "invalid sizes"),
                      (dict(a6=1 << 30), "invalid sizes"), (dict(a7=-1), "invalid sizes"), (dict(a0=None), "null pointer"),
                      (dict(a5=None), "null pointer"), (dict(a12=P + 8), "16-byte aligned")):
        assert match in refused("h3sa_fork_pages", pools, *changed(fork, **at))
    for at, match in ((dict(a1=-1), "invalid sizes"), (dict(a1=1 << 30), "invalid sizes"), (dict(a6=None), "null pointer"),
                      (dict(a7=P + 8), "16-byte aligned")):
        assert match in refused("h3sa_compact_pages", pools, *changed(compact, **at))
    for at, match in ((dict(a5=0), "invalid sizes"), (dict(a1=1 << 30), "invalid sizes"), (dict(a6=None), "null pointer")):
        assert match in refused("h3sa_free_pages", *changed(free, **at))
    for name, value, match in (("row_bytes", 24, "multiple of 16"), ("base", P + 8, "16-byte aligned"),
                               ("heads", 0, "invalid pools"), ("pages", 1 << 24, "too large")):
        broken = _lib.Pools()
        ctypes.pointer(broken)[0] = pools
        setattr(broken, name, value)
        assert match in refused("h3sa_fork_pages", broken, *fork)


def test_wrappers_take_cuda_tensors_only() -> None:
    from h3sa.branches import compact_pages, fork_pages, free_pages, shared_prefix_attention

    i = torch.zeros(1, 2, dtype=torch.int32)
    one, refs = i[:, 0].contiguous(), torch.zeros(2, dtype=torch.int32)
    pool = torch.zeros(1, 256, 128, dtype=torch.bfloat16)
    for call in (lambda: fork_pages([pool], i, one, refs, one), lambda: compact_pages([pool], i, refs),
                 lambda: free_pages(i, one, refs, one.bool()),
                 lambda: shared_prefix_attention(pool.view(1, 256, 1, 128), pool, pool, i, one, 0, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
