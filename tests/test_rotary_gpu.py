"""Rotary positions against the definition in 64 bits.

Tolerance: angles are whole turns off by under 2^-25, cosines and sines by 2^-22 with the functions' own
errors, products and sum by 2^-23 of |x| + |y|; then one rounding to the type, half a step of the result.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import drafts as od

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _check(shape, pairs, *, axes=1, kind="bf16", interleaved=False, factor=1.0, positions="i32", base=1e4, view=lambda t: t,
           out=None, in_place=False, seed=0):
    from h3sa.rotary import rotary_frequencies, rotate

    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen).to(TYPES[kind])
    frequencies = rotary_frequencies(2 * pairs // axes, base=base)[0].repeat(axes, 1) if pairs else torch.zeros(1, 0, dtype=torch.float64)
    rows = (*shape[:-2], axes)
    where = torch.from_numpy({"i32": lambda: rng.integers(-(1 << 31), 1 << 31, rows).astype(np.int32), "i64": lambda: rng.integers(0, 1 << 33, rows),
                              "near": lambda: rng.integers(0, 9000, rows).astype(np.int32), "f64": lambda: rng.uniform(-1e4, 1e4, rows)}[positions]())
    dx = view(x.cuda())
    target = dx if in_place else None if out is None else out(torch.full(shape, 3.0, dtype=x.dtype, device="cuda"))
    dw = where.cuda()
    got = rotate(dx, dw if axes > 1 else dw[..., 0].contiguous(), frequencies.cuda() if axes > 1 else frequencies[0].cuda(),
                 interleaved=interleaved, factor=factor, out=target)
    if target is not None:
        assert got.data_ptr() == target.data_ptr()
    want = od.rotate(x, where, frequencies, interleaved, factor)
    half = torch.finfo(x.dtype).eps / 2
    smallest = torch.finfo(x.dtype).smallest_normal * half
    tol = half * want.abs() + smallest + 2.0 ** -20 * abs(factor) * 2 * x.double().abs().amax(-1, keepdim=True) * (1 if pairs else 0)
    off = (got.double().cpu() - want).abs()
    assert (off <= tol).all(), float((off / tol.clamp(min=1e-300)).max())
    if 2 * pairs < shape[-1]:
        assert torch.equal(got.cpu()[..., 2 * pairs:], x[..., 2 * pairs:])  # behind the last pair
    return got


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape,pairs,axes,positions", [
    ((1, 1, 128), 64, 1, "i32"), ((57, 14, 64), 32, 1, "near"), ((3, 5, 7, 128), 48, 3, "f64"), ((2000, 3, 80), 36, 1, "i64"),
    ((33, 2, 72), 12, 3, "near"), ((19, 4, 256), 128, 1, "i32"), ((5, 3, 13), 6, 1, "near"), ((5, 3, 2), 1, 1, "near"), ((4, 2, 96), 0, 1, "near"),
    ((2, 300, 1, 128), 64, 1, "near"), ((7, 1, 1024), 512, 1, "near"), ((6, 2, 130), 20, 1, "near")])
def test_rotate(shape, pairs, axes, positions, interleaved, kind) -> None:
    _check(shape, pairs, axes=axes, kind=kind, interleaved=interleaved, positions=positions, factor=0.7)


def test_rotate_strides_and_in_place() -> None:
    def slice_of_merged(t):
        wide = torch.full((*t.shape[:-2], 3 * t.shape[-2], t.shape[-1]), 9.0, dtype=t.dtype, device=t.device)
        wide[..., t.shape[-2]:2 * t.shape[-2], :] = t
        return wide[..., t.shape[-2]:2 * t.shape[-2], :]

    def odd(t):
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
        wide[..., 3:] = t
        return wide[..., 3:]

    def heads_first(t):
        return t.transpose(-2, -3).contiguous().transpose(-2, -3)

    for kind in ("bf16", "fp32"):
        for interleaved in (False, True):
            for view in (slice_of_merged, odd, heads_first):
                _check((2, 9, 4, 128), 64, kind=kind, interleaved=interleaved, view=view)
                _check((2, 9, 4, 128), 32, kind=kind, interleaved=interleaved, view=view, in_place=True)
                _check((11, 4, 128), 64, kind=kind, interleaved=interleaved, out=view)


def test_a_broadcast_input_and_rows_beside_a_view_stay() -> None:
    from h3sa.rotary import rotary_frequencies, rotate

    f = rotary_frequencies(128)[0].cuda()
    x = torch.randn(1, 4, 128, device="cuda")
    at = torch.arange(9, device="cuda")
    assert torch.equal(rotate(x.expand(9, 4, 128), at, f), rotate(x.expand(9, 4, 128).contiguous(), at, f))
    wide = torch.full((9, 6, 128), 5.0, device="cuda")
    rotate(x.expand(9, 4, 128), at, f, out=wide[:, 1:5])
    assert (wide[:, 0] == 5).all() and (wide[:, 5] == 5).all()


def test_rotate_of_nothing() -> None:
    from h3sa.rotary import rotary_frequencies, rotate

    f = rotary_frequencies(128)[0].cuda()
    for shape in ((0, 4, 128), (5, 0, 128), (0, 3, 2, 128), (2, 0, 2, 128)):
        x = torch.zeros(shape, device="cuda").bfloat16()
        assert rotate(x, torch.zeros(shape[:-2], dtype=torch.int32, device="cuda"), f).shape == shape


def test_many_tokens_pass_32_bits() -> None:
    """A tensor of more than 2^31 elements: the last tokens are where they belong."""

    from h3sa.rotary import rotary_frequencies, rotate

    tokens, heads = (1 << 31) // (32 * 128) + 77, 32
    f = rotary_frequencies(128)[0].cuda()
    x = torch.ones(1, 1, 128, device="cuda").bfloat16().expand(tokens, heads, 128)
    at = torch.arange(tokens, dtype=torch.int32, device="cuda")
    out = rotate(x, at, f)
    want = rotate(x[-50:].contiguous(), at[-50:].contiguous(), f)
    assert torch.equal(out[-50:], want)


def test_gradient_is_the_opposite_rotation() -> None:
    """Against the formula's (R^T g) and against differences, in fp32."""

    from h3sa.rotary import rotary_frequencies, rotate

    gen = torch.Generator().manual_seed(1)
    x, g, d = (torch.randn(23, 3, 128, generator=gen).cuda() for _ in range(3))
    at = torch.randint(0, 5000, (23,), generator=gen).cuda()
    f = rotary_frequencies(96)[0].cuda()
    for interleaved in (False, True):
        turn = lambda t, p, i=interleaved: rotate(t, p, f, interleaved=i, factor=1.3)  # noqa: E731
        grad = turn(g, -at)
        # behind the last pair the factor is not applied, nor is it in the gradient
        want = od.rotate(g.cpu(), -at.cpu()[:, None], f.cpu()[None], interleaved, 1.3)
        assert (grad.double().cpu() - want).abs().max() <= 2.0 ** -19 * g.abs().max().double().cpu()
        # the map is linear, so any step will do; each of the 8832 products is off by under 2^-20 of the largest
        slope = ((turn(x + 0.5 * d, at) - turn(x - 0.5 * d, at)).double() * g.double()).sum()
        assert abs(float(slope - (grad.double() * d.double()).sum())) <= 8832 * 2.0 ** -20 * 25


def test_rotate_in_two_graphs_on_another_stream() -> None:
    from h3sa.rotary import rotary_frequencies, rotate

    f = rotary_frequencies(128)[0].cuda()
    x, at = torch.randn(40, 4, 128, device="cuda").bfloat16(), torch.arange(40, device="cuda")
    rotate(x, at, f)
    outs, graphs = [torch.empty_like(x) for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, out in zip(graphs, outs):
        with torch.cuda.graph(graph):
            rotate(x, at, f, out=out)
    at += 1000
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    got = rotate(x, at, f, stream=side)
    torch.cuda.synchronize()
    want = rotate(x, at, f)
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(got, want)
