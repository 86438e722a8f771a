"""Rotations in fp32, against angles in whole numbers.

u = 2^-24, half a step of a number of 1. A fraction of a turn has 32 bits, cut off (2^-32), of a frequency off by
2^-65 of a turn a position (2^-34 for any of 32 bits): 2^-29 of an angle. Its first 24 bits go through a function that is
off by one step of a result below 1, u; the rest is added by one multiply-add, u / 2. Together under 1.6 u. Then, of
(x, y) -> x c - y s: a factor not 1 is a rounding of c and s, u of each; y s is rounded once and so is the sum.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import angles

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _angles(kind: str, rng: np.random.Generator, tokens: int) -> tuple[torch.Tensor, np.ndarray, np.ndarray]:
    """Positions, whole numbers and frequencies with the same products, and the frequencies themselves."""

    from h3sa.rotary import rotary_frequencies

    frequencies = rotary_frequencies(64, base=1e4)[0].numpy()
    if kind == "f64":  # sixteenths, below 2^11 with what fp64 products of 53 bits leave: 2^-42
        whole = rng.integers(0, 1 << 15, tokens)
        return torch.from_numpy(whole / 16.0), whole, frequencies / 16.0
    whole = rng.integers(-(1 << 31), 1 << 31, tokens) if kind == "far" else rng.integers(0, 9000, tokens)
    return torch.from_numpy(whole.astype(np.int64 if kind == "i64" else np.int32)), whole, frequencies


@pytest.mark.parametrize("kind", ["near", "far", "i64", "f64"])
def test_cosines_and_sines(kind) -> None:
    """Rows of (1, 0), whose results are cosine and sine as they are."""

    from h3sa.rotary import rotate

    positions, whole, frequencies = _angles(kind, np.random.default_rng(1), 1500)
    x = torch.zeros(len(whole), 1, 64, device="cuda")
    x[..., :32] = 1.0
    frequency = torch.from_numpy(_angles(kind, np.random.default_rng(1), 1)[2]) * (16.0 if kind == "f64" else 1.0)
    got = rotate(x, positions.cuda(), frequency.cuda())[:, 0].double().cpu()
    for have, want in zip(got.chunk(2, dim=-1), angles.cos_sin(whole, frequencies)):
        off = (have - torch.from_numpy(want)).abs()
        assert off.max() <= 1.6 * U, float(off.max() / U)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["near", "far"])
@pytest.mark.parametrize("pad", [0, 3])  # vectors, single values
def test_rotations(kind, interleaved, pad) -> None:
    from h3sa.rotary import rotate

    gen, factor = torch.Generator().manual_seed(2), 0.7
    positions, whole, frequencies = _angles(kind, np.random.default_rng(2), 400)
    pairs = torch.randn(400, 3, 2, 32, generator=gen)
    x, y = pairs[:, :, 0].double(), pairs[:, :, 1].double()
    rows = pairs.transpose(-1, -2) if interleaved else pairs
    wide = torch.zeros(400, 3, 64 + pad, device="cuda")
    wide[..., pad:] = rows.reshape(400, 3, 64).cuda()
    out = rotate(wide[..., pad:], positions.cuda(), torch.from_numpy(frequencies).cuda(), interleaved=interleaved, factor=factor)
    got = out.double().cpu().view(400, 3, 32, 2).transpose(-1, -2) if interleaved else out.double().cpu().view(400, 3, 2, 32)
    c, s = (torch.from_numpy(t)[:, None] * float(np.float32(factor)) for t in angles.cos_sin(whole, frequencies))
    for have, want in zip(got.unbind(2), (x * c - y * s, x * s + y * c)):
        tol = factor * (x.abs() + y.abs()) * (1.6 + 1.0 + 1.0) * U + want.abs() * U
        off = (have - want).abs()
        assert (off <= tol).all(), float((off / tol).max())
