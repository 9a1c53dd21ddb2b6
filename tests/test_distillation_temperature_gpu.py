"""Distillation at temperatures whose square leaves fp32: the loss is T (T sum), of which neither factor does."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.distillation import TopKDistillation  # noqa: E402


def _row_loss(student, indices, temperature):
    rows, vocab = student.shape
    out = torch.empty(rows, device="cuda")
    TopKDistillation(rows, vocab, 1).run(logits=student, teacher_values=torch.zeros(rows, 1, device="cuda"), teacher_indices=indices,
                                         temperature=temperature, row_loss=out)
    return out


@pytest.mark.parametrize("vocab", [2, 300, 1000, 1500, 3000, 40000])
@pytest.mark.parametrize("temperature", [1e-30, 1e-25, 1e-21])
def test_low(vocab, temperature):
    """A teacher on a token 1 below all others: T^2 (1 / T + T ln(vocab - 1) ...) = T to fp32, 6 roundings."""
    student = torch.full((3, vocab), 1.0, device="cuda")
    student[:, 1] = 0.0
    indices = torch.ones(3, 1, dtype=torch.int32, device="cuda")
    t = float(torch.tensor(temperature))
    assert bool(((_row_loss(student, indices, temperature).double() - t).abs() <= 6 * 2.0 ** -24 * t + 2.0 ** -149).all())


@pytest.mark.parametrize("temperature", [2e19, 1e25, 1e30])
def test_high(temperature):
    """A single token: nothing to lose."""
    student, indices = torch.randn(3, 1, device="cuda"), torch.zeros(3, 1, dtype=torch.int32, device="cuda")
    assert not bool(_row_loss(student, indices, temperature).any())
