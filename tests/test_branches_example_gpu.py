"""The branch operators as an example program runs them: fork, write, attend, free, compact."""

import importlib.util
import pathlib

import pytest
import torch

pytestmark = pytest.mark.gpu

_PATH = pathlib.Path(__file__).resolve().parents[1] / "examples" / "branched_history.py"


def _example():
    spec = importlib.util.spec_from_file_location("branched_history", _PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


# A result is a convex combination of values, computed with P and the result in bf16: each rounds by
# at most 2^-8 of the largest value. The sum over P is of unrounded terms, hence one 2^-8 for P's
# numerator, and 2^-8 for the result; scores in fp32 add under 2^-12.
_TOLERANCE = 2 * 2.0 ** -8 + 2.0 ** -12


@pytest.mark.parametrize("history,branches,rows,steps", [
    (1000, 4, 16, 3),   # a partial page behind the shared ones
    (256, 3, 1, 2),     # whole pages, single rows
    (1, 2, 130, 2),     # nothing to share, new rows over page ends
    (640, 2, 200, 1),   # a branch's rows fill whole tiles
])
def test_rounds_of_branches(history, branches, rows, steps):
    worst = _example().run(history=history, branches=branches, rows=rows, steps=steps, check=True)
    assert worst <= _TOLERANCE
