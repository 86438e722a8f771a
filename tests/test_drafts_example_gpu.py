"""The operators of a drafting step as an example program runs them: tree, append, attend, keep, step after step."""

import importlib.util
import pathlib

import pytest

pytestmark = pytest.mark.gpu

_PATH = pathlib.Path(__file__).resolve().parents[1] / "examples" / "drafted_trees.py"


def _example():
    spec = importlib.util.spec_from_file_location("drafted_trees", _PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


# A result is a convex combination of values, with P and the result in bf16: each rounds by at most 2^-8 of
# the largest value, and fp32 scores add under 2^-12. A rotated key that the two sides round to different
# neighbours (2^-7 of it; fp32 products off by 2^-20 do that to one element in 2^11) moves a score by q k 2^-7 /
# sqrt(128) for that element, under 2^-7 here, and a weight by as much: far below 2^-9 of the result in all.
_TOLERANCE = 2 * 2.0 ** -8 + 2.0 ** -12 + 2.0 ** -9


@pytest.mark.parametrize("history,sequences,nodes,steps,heads", [
    (600, 4, 12, 4, 8),    # a partial page behind the shared ones
    (256, 3, 1, 3, 8),     # whole pages, single rows
    (130, 2, 40, 5, 12),   # trees of 240 stacked rows, paths over page ends
    (50, 3, 9, 2, 2),      # nothing shared
])
def test_steps_of_drafts(history, sequences, nodes, steps, heads):
    worst = _example().run(history=history, sequences=sequences, nodes=nodes, steps=steps, heads=heads, check=True)
    assert worst <= _TOLERANCE
