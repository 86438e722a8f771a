"""What the C entry points of drafted trees and rotary positions refuse before any launch, the frequencies against their
formulas, and the oracle against itself."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import drafts as od

P = 1 << 20  # a 16-byte aligned address that nothing dereferences
TOP = (1 << 31) - 1


def _lib():
    from h3sa import _lib

    return _lib


def _heads(**change):
    heads = _lib().Heads()
    for name, value in {**dict(base=P, stride_sequence=1024, stride_row=256, stride_head=128, heads=2), **change}.items():
        setattr(heads, name, value)
    return heads


def _rotary(**change):
    rotary = _lib().RotaryPositions()
    for name, value in {**dict(positions=P, frequencies=P, position_kind=1, axes=1, pairs=64, interleaved=0, factor=1.0), **change}.items():
        setattr(rotary, name, value)
    return rotary


def _refused(name: str, args, match: str) -> None:
    lib = _lib()
    code = getattr(lib.LIB, name)(*args)
    assert code in (lib.H3SA_ERR_INVALID, lib.H3SA_ERR_UNSUPPORTED) and match in lib.last_error(), (code, lib.last_error())


def _call(name: str, defaults: dict, change: dict, match: str) -> None:
    _refused(name, {**defaults, **change}.values(), match)


TREE = dict(parents=P, batch=2, nodes=9, lengths=P, counts=None, masks=P, positions=P, err=None, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(batch=-1), "invalid sizes"), (dict(nodes=-1), "invalid sizes"), (dict(nodes=1025), "invalid sizes"), (dict(batch=65536), "invalid sizes"),
    (dict(parents=None), "null pointer"), (dict(lengths=None), "null pointer"), (dict(masks=None), "null pointer"), (dict(positions=None), "null pointer"),
])
def test_tree_refuses(change, match) -> None:
    _call("h3sa_draft_tree", TREE, change, match)


@pytest.mark.parametrize("x,out,change,rotary,match", [
    ({}, {}, dict(batch=-1), {}, "invalid sizes"), ({}, {}, dict(rows=-1), {}, "invalid sizes"), ({}, {}, dict(dim=0), {}, "invalid sizes"),
    ({}, {}, dict(dim=1025), {}, "invalid sizes"), (dict(heads=3), {}, {}, {}, "invalid sizes"), ({}, {}, dict(dtype=3), {}, "unknown type"),
    ({}, {}, dict(dtype=-1), {}, "unknown type"), ({}, {}, {}, dict(pairs=65), "do not fit"), ({}, {}, {}, dict(pairs=-1), "do not fit"),
    ({}, {}, {}, dict(pairs=64, axes=3), "do not fit"), ({}, {}, {}, dict(axes=0), "do not fit"), ({}, {}, {}, dict(position_kind=4), "positions must be"),
    ({}, {}, {}, dict(position_kind=0), "positions must be"), ({}, {}, {}, dict(positions=None), "null pointer"), ({}, {}, {}, dict(frequencies=None), "null pointer"),
    ({}, {}, {}, dict(factor=math.inf), "finite"), ({}, {}, {}, dict(factor=math.nan), "finite"), (dict(base=None), {}, {}, {}, "null pointer"),
    ({}, dict(base=None), {}, {}, "null pointer"), (dict(base=P + 1), {}, {}, {}, "aligned"), ({}, dict(base=P + 2), dict(dtype=2), {}, "aligned"),
    ({}, dict(stride_head=0), {}, {}, "overlap"), ({}, dict(stride_row=127), {}, {}, "overlap"), ({}, dict(stride_sequence=-100), {}, {}, "overlap"),
    (dict(stride_head=1 << 31), {}, {}, {}, "32 bits"), ({}, dict(stride_head=-(1 << 31) - 1), {}, {}, "32 bits"),
    ({}, {}, dict(batch=1 << 20, rows=1 << 11), {}, "too large"), (dict(heads=1 << 12), dict(heads=1 << 12), dict(batch=1 << 10, rows=1 << 9), {}, "too large"),
])
def test_rotate_refuses(x, out, change, rotary, match) -> None:
    args = {**dict(x=_heads(**x), out=_heads(**out), dtype=0, batch=2, rows=4, dim=128, rotary=_rotary(**rotary), stream=None), **change}
    _refused("h3sa_rotate", args.values(), match)


APPEND = dict(key=None, value=None, query=None, query_out=None, batch=2, rows=4, k=P, v=P, pages=8, e4m3=0, ks=None, vs=None,
              table=P, width=4, lengths=P, counts=None, rotary=None, err=None, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(batch=-1), "invalid sizes"), (dict(rows=-1), "invalid sizes"), (dict(key=dict(heads=0), value=dict(heads=0)), "invalid sizes"),
    (dict(value=dict(heads=3)), "invalid sizes"), (dict(query={}), "invalid sizes"), (dict(query={}, query_out=dict(heads=3)), "invalid sizes"),
    (dict(pages=0), "invalid pool"), (dict(pages=1 << 24), "invalid pool"), (dict(width=0), "invalid pool"), (dict(width=1 << 24), "invalid pool"),
    (dict(k=None), "null pointer"), (dict(table=None), "null pointer"), (dict(lengths=None), "null pointer"), (dict(key=dict(base=None)), "null pointer"),
    (dict(query=dict(base=None), query_out={}), "null pointer"), (dict(e4m3=1, ks=P), "null pointer"), (dict(k=P + 8), "16-byte aligned"),
    (dict(key=dict(base=P + 1)), "aligned"), (dict(query={}, query_out=dict(base=P + 1)), "aligned"), (dict(value=dict(stride_head=1 << 31)), "32 bits"),
    (dict(batch=1 << 20, rows=1 << 11), "too large"), (dict(batch=1 << 14, rows=1 << 14), "too large"),
    (dict(query={}, query_out=dict(stride_row=0)), "overlap"), (dict(query={}, query_out=dict(stride_head=64)), "overlap"),
    (dict(rotary=dict(pairs=65)), "do not fit"), (dict(rotary=dict(position_kind=0, axes=2)), "positions must be"), (dict(rotary=dict(factor=-math.inf)), "finite"),
])
def test_append_refuses(change, match) -> None:
    args = {**APPEND, **dict(key={}, value={}), **change}
    for name in ("key", "value", "query", "query_out"):
        args[name] = None if args[name] is None else _heads(**args[name])
    args["rotary"] = None if args["rotary"] is None else _rotary(**args["rotary"])
    _refused("h3sa_append_rows", args.values(), match)


ATTEND = dict(q=P, sb=512, sn=512, sh=128, out=P, lse=None, batch=2, rows=1, heads=4, kv=2, k=P, v=P, pages=4, e4m3=0, ks=None,
              vs=None, table=P, width=4, lengths=P, masks=P, counts=None, shared=128, scale=0.1, work=P, bytes=1 << 40, err=None, stream=None)


@pytest.mark.parametrize("change,match", [
    (dict(masks=None), "masks are missing"), (dict(width=TOP // 128, pages=4, rows=TOP % 128 + 1), "too large"), (dict(heads=3), "multiple of kv_heads"),
    (dict(batch=-1), "invalid sizes"), (dict(pages=0), "invalid pool"), (dict(width=1 << 24), "invalid pool"), (dict(shared=64), "whole pages"),
    (dict(shared=5 * 128), "whole pages"), (dict(q=None), "null pointer"), (dict(work=None), "null pointer"), (dict(e4m3=1, ks=P), "null pointer"),
    (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(q=P + 8), "16-byte aligned"), (dict(sn=516), "16-byte aligned"),
    (dict(batch=1 << 20, rows=1 << 10), "too large"), (dict(batch=1 << 14, rows=64, width=1 << 16, pages=1 << 16), "work index"), (dict(bytes=64), "workspace of 64"),
])
def test_tree_attention_refuses(change, match) -> None:
    _call("h3sa_tree_attention", ATTEND, change, match)


def test_tree_workspace_of_what_is_refused_is_none() -> None:
    work = _lib().LIB.h3sa_tree_workspace
    good = [2, 9, 4, 2, 128, 4, 0]
    assert work(*good) > 0
    for i, bad in ((0, 0), (1, 0), (2, 3), (3, 0), (4, -128), (4, 5 * 128), (5, 0)):
        assert work(*[bad if j == i else x for j, x in enumerate(good)]) == 0


KEEP = dict(pools=None, table=P, sequences=2, width=4, lengths=P, path=P, steps=3, out=P, err=None, stream=None)


@pytest.mark.parametrize("pools,change,match", [
    (dict(row_bytes=24), {}, "row bytes"), (dict(row_bytes=1 << 24), {}, "row bytes"), (dict(pages=1 << 24), {}, "too large"), (dict(base=None), {}, "non-null"),
    (dict(base=P + 8), {}, "16-byte aligned"), (dict(count=0), {}, "none or too many"), (dict(heads=1 << 20), dict(sequences=1 << 12, width=1), "none or too many"),
    ({}, dict(sequences=-1), "invalid sizes"), ({}, dict(width=0), "invalid sizes"), ({}, dict(steps=-1), "invalid sizes"), ({}, dict(sequences=1 << 16, width=1, steps=1 << 16), "invalid sizes"),
    ({}, dict(sequences=1 << 11, width=1 << 20), "invalid sizes"), ({}, dict(table=None), "null pointer"), ({}, dict(lengths=None), "null pointer"),
    ({}, dict(path=None), "null pointer"), ({}, dict(out=None), "null pointer"),
])
def test_keep_refuses(pools, change, match) -> None:
    p = _lib().Pools()
    for name, value in {**dict(base=P, stride=4096, count=2, heads=1, pages=8, row_bytes=32), **pools}.items():
        setattr(p, name, value)
    _call("h3sa_keep_rows", {**KEEP, "pools": p}, change, match)


@pytest.mark.parametrize("at", [(P, 2 * P, P), (2 * P, 3 * P, P, 3 * P + 32752), (P + 16, P)])
def test_keep_refuses_pools_that_overlap(at) -> None:
    """Rows of a tensor that is given twice would move twice."""

    p, listed = _lib().Pools(), (ctypes.c_void_p * len(at))(*at)
    for name, value in dict(list=ctypes.addressof(listed), count=len(at), heads=1, pages=8, row_bytes=32).items():
        setattr(p, name, value)
    _call("h3sa_keep_rows", {**KEEP, "pools": p}, {}, "overlap")


@pytest.mark.parametrize("stride", [0, 32752, -32752])
def test_keep_refuses_strides_that_overlap(stride) -> None:
    p = _lib().Pools()
    for name, value in dict(base=P, stride=stride, count=2, heads=1, pages=8, row_bytes=32).items():
        setattr(p, name, value)
    _call("h3sa_keep_rows", {**KEEP, "pools": p}, {}, "overlap")


def test_the_structs_are_the_header_s() -> None:
    assert ctypes.sizeof(_lib().Heads) == 40 and ctypes.sizeof(_lib().RotaryPositions) == 40


def test_wrappers_want_cuda_tensors() -> None:
    from h3sa import drafts
    from h3sa.rotary import rotary_frequencies, rotate

    x, n = torch.zeros(1, 2, 2, 128).bfloat16(), torch.zeros(1, dtype=torch.int32)
    pool, table = torch.zeros(2, 128, 128).bfloat16(), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="require CUDA"):
        rotate(x, torch.zeros(1, 2, dtype=torch.int32), rotary_frequencies(128)[0])
    for call in (lambda: drafts.append_rows(x, x, pool, pool, table, n), lambda: drafts.draft_tree(table, n), lambda: drafts.keep_rows([pool], table, n, table),
                 lambda: drafts.tree_attention(x, pool, pool, table, n, torch.zeros(1, 2, 1, dtype=torch.int32), 0.1)):
        with pytest.raises(RuntimeError, match="require CUDA"):
            call()


# ------------------------------------------------------------------------------------ frequencies


def test_frequencies_are_the_formulas() -> None:
    from h3sa.rotary import rotary_frequencies

    plain, factor = rotary_frequencies(96, base=5e5)
    assert plain.dtype == torch.float64 and factor == 1.0
    for k in range(48):
        assert math.isclose(plain[k], 5e5 ** (-2 * k / 96), rel_tol=1e-14)
    assert torch.allclose(rotary_frequencies(96, base=5e5, scaling="linear", scale=4.0)[0], plain / 4, rtol=1e-15)
    ntk, factor = rotary_frequencies(96, base=5e5, scaling="ntk", scale=4.0)
    assert factor == 1.0 and ntk[0] == 1.0 and math.isclose(ntk[-1], plain[-1] / 4, rel_tol=1e-13)
    parts, factor = rotary_frequencies(128, base=1e4, scaling="parts", scale=16.0, trained_rows=4096, slow=1.0, fast=32.0)
    assert math.isclose(factor, 0.1 * math.log(16.0) + 1.0)
    for k, f in enumerate(parts):
        own = 1e4 ** (-2 * k / 128)
        turns = 4096 * own / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
        assert math.isclose(f, own * keep + own / 16.0 * (1.0 - keep), rel_tol=1e-13)
    assert parts[0] == 1.0 and math.isclose(parts[-1], 1e4 ** (-126 / 128) / 16, rel_tol=1e-13)


@pytest.mark.parametrize("args,change", [((0,), {}), ((7,), {}), ((-2,), {}), ((64,), dict(base=0.0)), ((64,), dict(base=math.inf)), ((64,), dict(scale=0.5)),
                                         ((64,), dict(scale=math.nan)), ((64,), dict(scaling="none of these")), ((64,), dict(scaling="parts")),
                                         ((64,), dict(scaling="parts", trained_rows=10, slow=2.0, fast=1.0)), ((2,), dict(scaling="ntk"))])
def test_frequencies_refuse(args, change) -> None:
    from h3sa.rotary import rotary_frequencies

    with pytest.raises(ValueError, match="rotary_frequencies"):
        rotary_frequencies(*args, **change)


# ------------------------------------------------------------------------------------ the oracle


def test_oracle_rotation_is_a_rotation() -> None:
    """Lengths of pairs stay, rotations add up, products depend on the distance of positions alone."""

    gen = torch.Generator().manual_seed(0)
    x, y = (torch.randn(5, 2, 64, generator=gen, dtype=torch.float64) for _ in range(2))
    f = torch.rand(1, 24, generator=gen, dtype=torch.float64)
    at = torch.arange(5)[:, None] * 3
    for interleaved in (False, True):
        turn = lambda t, p, i=interleaved: od.rotate(t, p, f, i)  # noqa: E731
        torch.testing.assert_close(turn(turn(x, at), -at), x)
        torch.testing.assert_close(turn(turn(x, at), at + 7), turn(x, 2 * at + 7))
        torch.testing.assert_close((turn(x, at) * turn(y, at + 4)).sum(-1), (turn(x, at * 0) * turn(y, at * 0 + 4)).sum(-1))
        assert torch.equal(turn(x, at)[..., 48:], x[..., 48:])
    order = torch.cat((torch.arange(0, 48, 2), torch.arange(1, 48, 2), torch.arange(48, 64)))
    torch.testing.assert_close(od.rotate(x, at, f, True)[..., order], od.rotate(x[..., order], at, f, False))


def test_oracle_trees_and_attention() -> None:
    from oracle import branches as ob

    parents = np.array([[-1, 0, 0, 1, -1, 4]])
    sees = od.ancestors(parents, np.array([6]))
    assert [list(np.flatnonzero(r)) for r in sees[0]] == [[0], [0, 1], [0, 2], [0, 1, 3], [4], [4, 5]]
    assert od.words(sees)[0, :, 0].tolist() == [1, 3, 5, 11, 16, 48]
    wide = np.zeros((1, 40), bool)
    wide[0, [31, 32]] = True
    assert od.words(wide).tolist() == [[-(1 << 31), 1]]
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(2, 5 * 128, 128, generator=gen, dtype=torch.float64) for _ in range(2))
    table, lengths = np.array([[4, 1, -1], [3, 0, 2]]), np.array([200, 256])
    q = torch.randn(2, 3, 4, 128, generator=gen, dtype=torch.float64)
    chain = np.tri(3, dtype=bool)[None].repeat(2, 0)
    a = od.attention(q, k, v, table, lengths, np.array([3, 3]), chain, 0.1)
    b = ob.attention(q, k, v, table, lengths + 3, 0.1, causal=True)
    for x, y in zip(a, b):
        torch.testing.assert_close(x, y)


def test_oracle_keep() -> None:
    pool = torch.arange(3 * 128.0).view(1, 3 * 128, 1)
    out, kept = od.keep(pool, np.array([[2, 0]]), np.array([126]), np.array([[1, 3, 4, -1, 9]]))
    assert kept.tolist() == [129]
    assert out[0, [2 * 128 + 126, 2 * 128 + 127, 0], 0].tolist() == [2 * 128 + 127, 1, 2]
    assert int((out != pool).sum()) == 3
