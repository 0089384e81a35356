"""Calls on tensors of a GPU that is not the current one are made with that GPU current."""

from __future__ import annotations

import contextlib

import pytest
import torch

from tklab import _hip


@pytest.mark.parametrize("current", [0, 1])
def test_call_on_selects_the_tensors_device(monkeypatch, current) -> None:
    events = []

    @contextlib.contextmanager
    def selected(device):
        events.append(("select", device))
        yield
        events.append(("restore", device))

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current)
    monkeypatch.setattr(torch.cuda, "device", selected)
    monkeypatch.setitem(_hip._bound, "tk_rotary", lambda *args: events.append(args) or 0)
    _hip.call_on(1, "tk_rotary", 4, 2)
    assert events == ([(4, 2)] if current == 1 else [("select", 1), (4, 2), ("restore", 1)])


@pytest.mark.parametrize("current", [0, 1])
def test_call_on_raises_for_a_failed_call(monkeypatch, current) -> None:
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: current)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    monkeypatch.setitem(_hip._bound, "tk_rotary", lambda *args: 1)
    with pytest.raises(_hip.HipLibraryError, match="tk_rotary failed"):
        _hip.call_on(1, "tk_rotary", 4, 2)


def test_row_layout_packs_strides_and_refuses_rows_the_kernels_cannot_read() -> None:
    x = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    address, strides = _hip.row_layout(x, "x", -1)
    assert address == x.data_ptr() and strides == _hip.int64_bytes((768, 256, 64))
    assert list(memoryview(strides).cast("q")) == [768, 256, 64]
    with pytest.raises(ValueError, match="x must be on"):
        _hip.row_layout(x, "x", 0)
    with pytest.raises(ValueError, match="contiguous final"):
        _hip.row_layout(x.transpose(2, 3), "x", -1)
    with pytest.raises(ValueError, match="16-byte aligned"):
        _hip.row_layout(x[..., 1:], "x", -1)
    with pytest.raises(ValueError, match="16-byte aligned"):
        _hip.row_layout(torch.zeros(2, 3, 4, 60, dtype=torch.bfloat16), "x", -1)


def test_row_layout_takes_any_stride_of_a_single_entry() -> None:
    x = torch.zeros(4096, dtype=torch.bfloat16)
    one = x.as_strided((1, 3, 1, 64), (1027, 128, 2 ** 24 + 8, 1))
    address, strides = _hip.row_layout(one, "x", -1)
    batch, head, row = memoryview(strides).cast("q")
    assert address == x.data_ptr() and head == 128
    assert batch % 8 == 0 and row % 8 == 0 and 0 <= batch < 2 ** 24 and 64 <= row < 2 ** 24
    with pytest.raises(ValueError, match="16-byte aligned"):
        _hip.row_layout(x.as_strided((1, 3, 1, 64), (1027, 127, 5, 1)), "x", -1)
