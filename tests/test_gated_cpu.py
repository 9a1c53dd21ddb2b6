"""Gated feed-forward block without a GPU: the C entries refuse bad arguments with a message, and the
formulas that the GPU tests compare with agree with finite differences."""

import ctypes

import pytest
import torch

from robolearn_b200 import _native as N
from tests.test_gated_gpu import act64


def _error():
    return N.load().rl2_last_error().decode()


@pytest.mark.parametrize("desc,message", [
    ((0, 16, 16, 0, 0), "must be positive"),
    ((4, -1, 16, 0, 0), "must be positive"),
    ((4, 16, 1 << 25, 0, 0), "must be positive"),
    ((4, 16, 16, 2, 0), "dtype must be"),
    ((4, 16, 16, 0, 3), "activation"),
])
def test_create_refuses(desc, message):
    lib = N.load()
    assert lib.rl2_gated_create(ctypes.byref(N.GatedDesc(*desc))) is None
    assert message in _error()


def test_null_arguments():
    lib = N.load()
    assert lib.rl2_gated_create(None) is None
    assert lib.rl2_gated_workspace_bytes(None) == -1
    assert lib.rl2_gated_forward(None, None, None) == -1 and "null" in _error()
    assert lib.rl2_gated_backward(None, None, None) == -1 and "null" in _error()
    assert lib.rl2_gated_forward(None, ctypes.byref(N.GatedForwardArgs(rows=1)), None) == -1 and "null" in _error()
    assert lib.rl2_gated_destroy(None) == 0


@pytest.mark.parametrize("name", ["silu", "gelu", "relu"])
def test_slopes_against_differences(name):
    g = torch.linspace(-6, 6, 97, dtype=torch.float64) + 1e-3  # away from ReLU's kink
    eps = 1e-6
    numeric = (act64(name, g + eps)[0] - act64(name, g - eps)[0]) / (2 * eps)
    assert torch.allclose(act64(name, g)[1], numeric, atol=1e-9)
