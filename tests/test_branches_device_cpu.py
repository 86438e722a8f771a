"""A call's tensors lie on the current device, and so does its stream: a kernel launched elsewhere would be
given another GPU's addresses. Devices are stand-ins here."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch


def test_handle_refuses_another_device(monkeypatch) -> None:
    from h3sa import branches

    here, there = torch.device("cuda", 0), torch.device("cuda", 1)
    monkeypatch.setattr(branches, "_current_device", lambda: 0)
    monkeypatch.setattr(branches, "_raw_stream", lambda index: 40 + index)
    assert branches._handle(None, here) == 40
    assert branches._handle(SimpleNamespace(device=here, cuda_stream=7), here) == 7
    for stream, device in ((None, there), (SimpleNamespace(device=there, cuda_stream=7), here),
                           (SimpleNamespace(device=there, cuda_stream=7), there),
                           (SimpleNamespace(device=here, cuda_stream=7), there)):
        with pytest.raises(RuntimeError, match="current device"):
            branches._handle(stream, device)
