"""Arguments that a 32-bit parameter of the C entry points would cut short."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _z(*shape, dtype=torch.int32):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


@pytest.mark.parametrize("shared_rows", [1 << 32, (1 << 32) + 128, -(1 << 32), (1 << 31) + (1 << 32)])
def test_shared_rows_past_32_bits(shared_rows) -> None:
    from h3sa.branches import shared_prefix_attention

    k = _z(2, 256, 128, dtype=torch.bfloat16)
    q = _z(1, 1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="whole pages"):
        shared_prefix_attention(q, k, k, _z(1, 2), _z(1), shared_rows, 1.0)


@pytest.mark.parametrize("reserve_rows", [1 << 31, 1 << 32, (1 << 32) + 1])
def test_reserve_rows_past_32_bits(reserve_rows) -> None:
    from h3sa.branches import fork_pages

    with pytest.raises(ValueError, match="reserve_rows"):
        fork_pages(_z(1, 1, 256, 8, dtype=torch.float32), _z(1, 2), _z(1), _z(2), _z(1), reserve_rows=reserve_rows)
