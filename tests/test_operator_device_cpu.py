"""Operators of policies over discrete tokens refuse a call while another device is current, or on another device's
stream: their launches would go to the current device with the other's addresses. On the host: the query of the current
device is replaced, CPU tensors stand for the operator's, and nothing may reach the library."""

from types import SimpleNamespace

import pytest
import torch

from robolearn_b200 import _native as N
from robolearn_b200.distillation import TopKDistillation
from robolearn_b200.gated import GatedMLP
from robolearn_b200.token_sampling import TokenSampler

HERE = torch.zeros(1).get_device()  # index of the CPU tensors' device


class _Library:
    """Counts what reaches it."""

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def call(*args):
            self.calls += 1
            return 0

        return call


class _Stream(SimpleNamespace):
    def wait_stream(self, other):
        raise AssertionError("nothing is enqueued by a refused call")


def _operator(cls, **fields):
    op = object.__new__(cls)
    for name, value in dict(device=SimpleNamespace(index=HERE), _lib=_Library(), handle=None, **fields).items():
        setattr(op, name, value)
    return op


def _sampler(stream=None):
    op = _operator(TokenSampler, rows=3, vocab=8)
    op.run(logits=torch.zeros(3, 8), uniforms=torch.zeros(3), tokens=torch.zeros(3, dtype=torch.int32), stream=stream)
    return op


def _distillation(stream=None):
    op = _operator(TopKDistillation, rows=3, vocab=8, top=2, counter=torch.zeros(1, dtype=torch.int32), row_loss=torch.zeros(3))
    op._counter = op.counter.data_ptr()
    op.run(logits=torch.zeros(3, 8), teacher_values=torch.zeros(3, 2), teacher_indices=torch.zeros(3, 2, dtype=torch.int32), stream=stream)
    return op


def _gated(stream=None):
    op = _operator(GatedMLP, rows=3, features=8, hidden=8, dtype=torch.float16, _types=(torch.float16,))
    x = torch.zeros(3, 8, dtype=torch.float16)
    w = torch.zeros(8, 8, dtype=torch.float16)
    op.forward(x=x, gate_weight=w, up_weight=w, out=x.clone(), stream=stream)
    return op


@pytest.mark.parametrize("call", [_sampler, _distillation, _gated])
def test_another_device_is_current(call, monkeypatch):
    library = _Library()
    monkeypatch.setattr(f"{__name__}._Library", lambda: library)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: HERE + 1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 0, raising=False)
    with pytest.raises(ValueError, match="current device"):
        call()
    with pytest.raises(ValueError, match="current device"):
        call(_Stream(device_index=HERE, cuda_stream=64))
    assert library.calls == 0


@pytest.mark.parametrize("call", [_sampler, _distillation, _gated])
def test_stream_of_another_device(call, monkeypatch):
    library = _Library()
    monkeypatch.setattr(f"{__name__}._Library", lambda: library)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: HERE, raising=False)
    with pytest.raises(ValueError, match="stream must be of"):
        call(_Stream(device_index=HERE + 1, cuda_stream=64))
    assert library.calls == 0


def test_the_device_itself(monkeypatch):
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    assert N.raw_stream(None, 1) == 101
    assert N.raw_stream(_Stream(device_index=1, cuda_stream=64), 1) == 64
