"""Inputs on a device that is not the current one, without a second GPU: the launch happens with the inputs' device current, and
inputs on two devices are refused."""
import contextlib

import pytest
import torch


class On:
    """stands for a tensor: what the entry points ask before they launch"""

    def __init__(self, device, *shape):
        self.device, self.shape, self.is_cuda = torch.device(device), shape, True

    def dim(self):
        return len(self.shape)

    def float(self):
        return self


def gate(monkeypatch, made, other):
    from vc3d import scan
    monkeypatch.setattr(scan._GateProjectionFn, "apply", lambda *a: made())
    return lambda: scan.gate_projection(On("cuda:1", 4, 64), On("cuda:1", 128, 64), On(other, 128), None)


def lstm(monkeypatch, made, other):
    from vc3d import lstm
    monkeypatch.setattr(lstm._LSTMCellFn, "apply", lambda *a: made())
    one = On("cuda:1", 4, 64)
    return lambda: lstm.lstm_cell(one, one, one, one, one, one, On(other, 4, 64), None)


@pytest.mark.parametrize("entry", [gate, lstm])
def test_launches_with_the_inputs_device_current(entry, monkeypatch):
    from vc3d import ops
    from vc3d.capi import Vc3dError
    current = [0]

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d.index
        yield
        current[0] = before
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    assert entry(monkeypatch, lambda: current[0], "cuda:1")() == 1 and current[0] == 0
    current[0] = 1
    assert entry(monkeypatch, lambda: current[0], "cuda:1")() == 1 and current[0] == 1
    with pytest.raises(Vc3dError):
        entry(monkeypatch, lambda: None, "cuda:0")()
