"""Rotary positions of any tensor of heads.

``rotate`` turns pair k of each head by ``position * frequencies[k]``: pairs in halves ``(k, k + pairs)`` or
interleaved ``(2k, 2k + 1)``, over the first ``2 * pairs`` dimensions, the others staying as they are.
``rotary_frequencies`` makes the frequencies, for long contexts too. Angles are taken in 64 bits, so
positions may lie far out or between whole numbers, and results are rounded once. (The prologue of the
reference's processor, ``h3sa.prologue``, has a bf16 table of cosines and sines instead and rounds where the
reference does.) ``h3sa.drafts.append_rows`` takes the same frequencies.

A rotation's gradient is the rotation by the opposite angle: ``rotate(grad, -positions, ...)``, which also
takes a key from one position to another.
"""

from __future__ import annotations

import math

import torch

from ._lib import LIB, Heads, RotaryPositions, check
from .branches import _handle, _on

_ROTATE = LIB.h3sa_rotate
_F64 = torch.float64
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POSITIONS = {torch.int32: 1, torch.int64: 2, torch.float64: 3}
_empty_like = torch.empty_like


def rotary_frequencies(dim: int, *, base: float = 10000.0, scaling: str = "none", scale: float = 1.0,
                       trained_rows: int = 0, slow: float = 1.0, fast: float = 32.0,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """``(frequencies, factor)`` of ``dim`` rotated dimensions: fp64 ``[dim / 2]``, radians a position.

    ``scaling`` for contexts ``scale`` times as long as the trained ones:

    * ``"none"``: f_k = base^(-2k / dim);
    * ``"linear"``: f_k / scale (positions pressed together);
    * ``"ntk"``: base * scale^(dim / (dim - 2)) for base, which leaves f_0 and divides the last by ``scale``;
    * ``"parts"``: f_k where a pair makes more than ``fast`` turns in ``trained_rows`` positions, f_k /
      scale below ``slow``, a linear mix between, and factor 1 + 0.1 ln(scale) on queries and keys alike
      (YaRN, Peng et al. 2023).

    Several axes: ``frequencies.repeat(axes, 1)`` of ``dim / axes`` dimensions each.
    """

    if dim <= 0 or dim % 2:
        raise ValueError(f"rotary_frequencies: {dim} dimensions are no whole pairs")
    if not base > 0.0 or not scale >= 1.0 or math.isinf(base) or math.isinf(scale):
        raise ValueError("rotary_frequencies: base must be positive, scale at least 1, both finite")
    k = torch.arange(dim // 2, dtype=_F64)
    if scaling == "ntk":
        if dim < 4:
            raise ValueError("rotary_frequencies: \"ntk\" needs two pairs")
        base = base * scale ** (dim / (dim - 2))
    f = base ** (-2.0 * k / dim)
    factor = 1.0
    if scaling == "linear":
        f = f / scale
    elif scaling == "parts":
        if trained_rows <= 0 or not 0.0 <= slow < fast:
            raise ValueError("rotary_frequencies: \"parts\" needs trained_rows and 0 <= slow < fast")
        keep = ((trained_rows * f / (2.0 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f / scale * (1.0 - keep) + f * keep
        factor = 1.0 + 0.1 * math.log(scale)
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"rotary_frequencies: unknown scaling {scaling!r}")
    return f.to(device), factor


def _rotary(what: str, frequencies: torch.Tensor, positions: torch.Tensor | None, rows: tuple[int, ...], dim: int,
            interleaved: bool, factor: float, device: torch.device) -> RotaryPositions:
    """The rotation of rows of the given shape; without positions, a row's place in its sequence."""

    if frequencies.dtype is not _F64 or frequencies.device != device or not frequencies.is_contiguous():
        raise RuntimeError(f"{what}: frequencies must be contiguous float64 on {device}")
    if frequencies.ndim not in (1, 2):
        raise RuntimeError(f"{what}: frequencies must be [pairs] or [axes, pairs of an axis]")
    pairs, axes = frequencies.numel(), 1 if frequencies.ndim == 1 else frequencies.shape[0]
    if 2 * pairs > dim:
        raise RuntimeError(f"{what}: {pairs} pairs do not fit a head of {dim}")
    if positions is None:
        if axes > 1:
            raise RuntimeError(f"{what}: {axes} axes need positions")
        return RotaryPositions(None, frequencies.data_ptr(), 0, 1, pairs, interleaved, factor, 0)
    shape, kind = positions.shape, _POSITIONS.get(positions.dtype)
    if kind is None or positions.device != device or not positions.is_contiguous():
        raise RuntimeError(f"{what}: positions must be contiguous int32, int64 or float64 on {device}")
    if shape != (*rows, axes) and (axes > 1 or shape != rows):
        raise RuntimeError(f"{what}: positions must be {[*rows]}" + (f" with {axes} axes each" if axes > 1 else ""))
    return RotaryPositions(positions.data_ptr(), frequencies.data_ptr(), kind, axes if pairs else 1, pairs, interleaved,
                           factor, 0)


def rotate(x: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *, interleaved: bool = False,
           factor: float = 1.0, out: torch.Tensor | None = None,
           stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """``x`` with its heads rotated, times ``factor`` where they are.

    ``x``: bf16, fp16 or fp32 ``[tokens, heads, dim]`` or ``[sequences, rows, heads, dim]``, ``dim`` up to 1024, any
    strides with contiguous rows (16 bytes are read at a time where pairs, ``dim``, strides and addresses
    are multiples of that). ``positions``: int32, int64 or float64, one a row, or ``[..., axes]``.
    ``frequencies``: fp64 ``[pairs]``, or ``[axes, pairs of an axis]``, where the pairs of the first axis come
    first. Both are finite, and an angle (int positions: a frequency) is below 2^50. ``out``: a tensor like ``x`` for
    the result, ``x`` itself for a rotation in place; it may not overlap ``x`` otherwise, nor its rows each other (an axis of
    ``out`` steps over all that those of smaller steps reach, as in slices and transposed views).
    """

    what = "rotate"
    if not x.is_cuda:
        raise RuntimeError("h3sa kernels require CUDA tensors")
    device, shape, kind = x.device, x.shape, _DTYPES.get(x.dtype)
    if kind is None or len(shape) not in (3, 4):
        raise RuntimeError(f"{what}: x must be bf16, fp16 or fp32 [tokens, heads, dim] or [sequences, rows, heads, dim]")
    if len(shape) == 3:
        batch, (rows, heads, dim), sb, (sn, sh, last) = 1, shape, 0, x.stride()
    else:
        (batch, rows, heads, dim), (sb, sn, sh, last) = shape, x.stride()
    rotary = _rotary(what, frequencies, positions, shape[:-2], dim, interleaved, factor, device)
    if last != 1:
        raise RuntimeError(f"{what}: rows of x must be contiguous")
    handle = _handle(stream, device)
    if out is None:
        with _on(stream):
            out = _empty_like(x) if x.is_contiguous() else x.new_empty(shape)
    elif out.dtype is not x.dtype or out.shape != shape or out.device != device or out.stride(-1) != 1:
        raise RuntimeError(f"{what}: out must be {x.dtype} {list(shape)} on {device} with contiguous rows")
    dn, dh, _ = out.stride()[-3:]
    code = _ROTATE(Heads(x.data_ptr(), sb, sn, sh, heads, 0),
                   Heads(out.data_ptr(), out.stride(0) if batch > 1 else 0, dn, dh, heads, 0), kind, batch, rows, dim,
                   rotary, handle)
    if code:
        check("h3sa_rotate", code)
    return out


__all__ = ["rotary_frequencies", "rotate"]
