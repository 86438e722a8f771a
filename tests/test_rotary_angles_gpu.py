"""Cosines and sines of a rotation, read off rows of (1, 0) pairs, against angles in whole numbers.

Tolerance: the fraction of a turn is off by under 2^-25, 2^-22.3 of an angle, cosine and sine of it by another 2^-23 (two
steps of 2^-24 of numbers below 1) and fp32 results of such rows are not rounded again: 2^-21 in all.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import angles

pytestmark = pytest.mark.gpu

# Whose remainder behind 32 bits of a turn is a tie of the first rounding, to within 2^-63, and ordinary ones beside them.
TIES = np.array([0.9319518373176483, 1.4125622233893529, 1.087249648357686, 0.9319518373176484, 1.0, 1e-4])
POSITIONS = {torch.int32: [0, 1, -1, 40, 9999, 100000, -77777, 1 << 20, (1 << 31) - 1, -(1 << 31)],
             torch.int64: [0, 3, 100000, (1 << 31) + 7, -(1 << 33), 1 << 36]}


def _turned(positions: torch.Tensor, frequencies: np.ndarray) -> tuple[torch.Tensor, torch.Tensor]:
    from h3sa.rotary import rotate

    x = torch.zeros(len(positions), 1, 2 * len(frequencies), device="cuda")
    x[..., :len(frequencies)] = 1.0
    out = rotate(x, positions.cuda(), torch.from_numpy(frequencies).cuda())[:, 0].double().cpu()
    return out.chunk(2, dim=-1)


def _check(positions: list[int], dtype: torch.dtype, frequencies: np.ndarray, tol: float) -> None:
    got = _turned(torch.tensor(positions, dtype=dtype), frequencies)
    for have, want in zip(got, angles.cos_sin(np.array(positions, dtype=object), frequencies)):
        off = (have - torch.from_numpy(want)).abs()
        assert off.max() <= tol, (float(off.max()), np.unravel_index(int(off.argmax()), off.shape))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_frequencies_at_a_tie(dtype) -> None:
    _check(POSITIONS[dtype], dtype, TIES, 2.0 ** -21)
    _check(POSITIONS[dtype], dtype, -TIES, 2.0 ** -21)


def test_frequencies_at_a_tie_at_rows_own_places() -> None:
    """Appended behind 10^8 rows, all of whose pages are the same one: bf16 keys, off by half a step more, 2^-9 of at
    most 1."""

    from h3sa.drafts import append_rows

    width, length = 800000, 100_000_000
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    key = torch.zeros(1, 3, 1, 128, device="cuda").bfloat16()
    key[..., :len(TIES)] = 1.0
    pools = [torch.zeros(1, 128, 128, device="cuda").bfloat16() for _ in range(2)]
    append_rows(key, key, *pools, table, torch.tensor([length], dtype=torch.int32, device="cuda"),
                frequencies=torch.from_numpy(TIES).cuda())
    cos, sin = angles.cos_sin(length + np.arange(3), TIES)
    for i in range(3):
        row = pools[0][0, (length + i) % 128].double().cpu()
        for have, want in ((row[:len(TIES)], cos[i]), (row[len(TIES):2 * len(TIES)], sin[i])):
            assert (have - torch.from_numpy(want)).abs().max() <= 2.0 ** -9 + 2.0 ** -20


def test_large_frequencies() -> None:
    """Up to 2^48 radians a position, where the product with 1 / (2 pi) takes more than the 32 bits behind those of a turn."""

    rng = np.random.default_rng(0)
    frequencies = rng.choice([-1.0, 1.0], 64) * rng.uniform(1.0, 2.0, 64) * 2.0 ** rng.integers(10, 48, 64)
    _check([0, 1, -3, 1000], torch.int32, frequencies, 2.0 ** -21)
    _check([1, 77777, -(1 << 31)], torch.int64, frequencies[np.abs(frequencies) < 2.0 ** 40], 2.0 ** -21)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_16_bit_rows(kind, interleaved) -> None:
    """The angle as a float of up to pi: 2^-26 of a turn, the float 2 pi and a product, together 2^-21.7; the approximate
    functions 2^-21.2: under 2^-20.3 of |x| + |y|. A factor, a product and the sum in 32 bits, 2^-24 each, leave it below
    2^-20; then half a step of the result."""

    from h3sa.rotary import rotary_frequencies, rotate

    rng, gen, factor = np.random.default_rng(3), torch.Generator().manual_seed(3), 1.25
    frequencies = rotary_frequencies(96, base=1e6)[0].numpy()
    positions = rng.integers(-(1 << 31), 1 << 31, 300).astype(np.int32)
    pairs = torch.randn(300, 5, 2, 48, generator=gen).to(kind)
    rows = (pairs.transpose(-1, -2) if interleaved else pairs).reshape(300, 5, 96)
    out = rotate(rows.cuda(), torch.from_numpy(positions).cuda(), torch.from_numpy(frequencies).cuda(), interleaved=interleaved, factor=factor)
    got = out.double().cpu().view(300, 5, 48, 2).transpose(-1, -2) if interleaved else out.double().cpu().view(300, 5, 2, 48)
    x, y = pairs.double().unbind(2)
    c, s = (torch.from_numpy(t)[:, None] * factor for t in angles.cos_sin(positions, frequencies))
    half = torch.finfo(kind).eps / 2
    for have, want in zip(got.unbind(2), (x * c - y * s, x * s + y * c)):
        slack = 2.0 ** -20 * factor * (x.abs() + y.abs())
        tol = slack + half * (want.abs() + slack) + half * torch.finfo(kind).smallest_normal
        assert ((have - want).abs() <= tol).all(), float(((have - want).abs() / tol).max())
