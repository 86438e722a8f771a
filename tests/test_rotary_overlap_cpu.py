"""Rows of a result that overlap are refused before any launch, also where no single stride says so."""

from __future__ import annotations

import pytest

P = 1 << 20  # a 16-byte aligned address that nothing dereferences


def _lib():
    from h3sa import _lib

    return _lib


def _heads(sequence: int, row: int, head: int, heads: int):
    return _lib().Heads(P, sequence, row, head, heads, 0)


# strides of sequences, rows and heads of 2 sequences x 4 rows x 2 heads of 128
OVERLAP = [(2048, 128, 128), (2048, 256, 256), (256, 256, 128), (512, 256, 128), (1023, 256, 128), (1024, 255, 128), (2048, 300, 512), (-512, 256, 128),
           (1024, -192, 128), (-(1 << 63), 0, 128)]
APART = [(1024, 256, 128), (512, 128, 1024), (128, 512, 256), (5000, 1000, 333), (-1024, 256, 128), (1024, 256, -128), (-(1 << 63), 256, 128)]


@pytest.mark.parametrize("strides", OVERLAP)
def test_rows_that_overlap_are_refused(strides) -> None:
    lib = _lib()
    rotary = lib.RotaryPositions(P, P, 1, 1, 64, 0, 1.0, 0)
    out = _heads(*strides, 2)
    code = lib.LIB.h3sa_rotate(_heads(1024, 256, 128, 2), out, 0, 2, 4, 128, rotary, None)
    assert code == lib.H3SA_ERR_INVALID and "overlap" in lib.last_error()
    key = _heads(1024, 256, 128, 2)
    code = lib.LIB.h3sa_append_rows(key, key, key, out, 2, 4, P, P, 8, 0, None, None, P, 4, P, None, None, None, None)
    assert code == lib.H3SA_ERR_INVALID and "overlap" in lib.last_error()


@pytest.mark.parametrize("strides", APART)
def test_rows_that_lie_apart_are_not(strides) -> None:
    """They get as far as the next check: an address of no whole elements."""

    lib = _lib()
    rotary = lib.RotaryPositions(P, P, 1, 1, 64, 0, 1.0, 0)
    out = lib.Heads(P + 1, *strides, 2, 0)
    code = lib.LIB.h3sa_rotate(_heads(1024, 256, 128, 2), out, 0, 2, 4, 128, rotary, None)
    assert code == lib.H3SA_ERR_INVALID and "aligned" in lib.last_error()


def test_an_axis_of_one_has_any_stride() -> None:
    lib = _lib()
    rotary = lib.RotaryPositions(P, P, 1, 1, 64, 0, 1.0, 0)
    out = lib.Heads(P + 1, 0, 0, 128, 2, 0)
    code = lib.LIB.h3sa_rotate(_heads(0, 256, 128, 2), out, 0, 1, 1, 128, rotary, None)
    assert code == lib.H3SA_ERR_INVALID and "aligned" in lib.last_error()
