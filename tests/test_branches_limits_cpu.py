"""Sizes at the ends of 32 bits: what the ledger's entry points refuse before any launch, so that no index
of a kernel passes 2^31."""

from __future__ import annotations

import ctypes

import pytest

P = 1 << 20  # a 16-byte aligned address that nothing dereferences
TOP = (1 << 31) - 1


def _pools(**change):
    from h3sa import _lib

    pools = _lib.Pools()
    for name, value in {**dict(base=P, stride=4096, count=1, heads=1, pages=8, row_bytes=32), **change}.items():
        setattr(pools, name, value)
    return pools


def _refused(fn: str, *args) -> str:
    from h3sa import _lib

    code = getattr(_lib.LIB, fn)(*args)
    assert code == _lib.H3SA_ERR_INVALID, (code, _lib.last_error())
    return _lib.last_error()


def _fork(pools=None, sequences=2, width=4, children=2, reserve=0):
    return "h3sa_fork_pages", pools or _pools(), P, sequences, width, P, P, P, children, reserve, 0, P, P, P, P, None, None


def _compact(pools=None, sequences=2, width=4):
    return "h3sa_compact_pages", pools or _pools(), P, sequences, width, P, P, P, P, P, None, None


def _free(sequences=2, width=4, pages=8):
    return "h3sa_free_pages", P, sequences, width, P, P, pages, P, P, P, P, None, None


@pytest.mark.parametrize("call", [
    _fork(sequences=TOP, width=1), _fork(children=TOP, width=1), _fork(sequences=1 << 11, width=1 << 20),
    _compact(sequences=TOP, width=1), _compact(sequences=TOP - 4000, width=1), _compact(sequences=1, width=1 << 24),
    _free(sequences=TOP, width=1), _free(sequences=TOP - 100, width=1), _free(sequences=1, width=TOP),
    _free(sequences=1, width=1 << 24), _free(pages=TOP), _free(pages=1 << 24),
], ids=lambda c: f"{c[0]}-{c[3] if c[0] != 'h3sa_free_pages' else c[2]}")
def test_tables_and_counts_past_the_index_are_refused(call) -> None:
    assert "invalid sizes" in _refused(*call)


@pytest.mark.parametrize("row_bytes", [1 << 24, (1 << 24) + 16, 1 << 28, (1 << 31) - 16])
def test_rows_whose_page_passes_32_bits_are_refused(row_bytes) -> None:
    for call in (_fork, _compact):
        name, *args = call(_pools(row_bytes=row_bytes))
        assert "row bytes" in _refused(name, *args)


def test_the_struct_is_the_header_s() -> None:
    from h3sa import _lib

    assert ctypes.sizeof(_lib.Pools) == 40
