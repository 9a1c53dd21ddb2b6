"""The distillation's total is a mean of the rows' losses also where their sum is more than fp32 holds."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.distillation import TopKDistillation  # noqa: E402
from tests.test_distillation_gpu import run  # noqa: E402


@pytest.mark.parametrize("rows", [8, 1100])
@pytest.mark.parametrize("vocab", [50, 700, 1500, 3000, 40000])
def test_mean_of_large_losses(rows, vocab):
    """A teacher on a token whose logit is 1e38 below the others: a loss of about 1e38 in every row."""
    student = torch.zeros(rows, vocab, device="cuda")
    indices = (torch.arange(rows, device="cuda") % vocab)[:, None].contiguous()
    student.scatter_(1, indices, -1e38)
    values = torch.zeros(rows, 1, device="cuda")
    for temperature in (1.0, 2.0):
        row_loss, loss = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda")
        TopKDistillation(rows, vocab, 1).run(logits=student, teacher_values=values, teacher_indices=indices, temperature=temperature,
                                             loss_weight=1.0 / rows, row_loss=row_loss, loss_out=loss)
        # T^2 (1e38 / T): one rounding each of scale, product, back to natural logarithms, T^2, and of the sums' terms
        want = temperature * float(student[0, 0].abs())
        assert abs(row_loss.double() - want).max().item() <= 8 * 2.0 ** -24 * want
        assert abs(loss.item() - want) <= (16 + rows / 32) * 2.0 ** -24 * want


def test_weights_of_rows():
    """Ordinary losses, weights that add up to no power of two."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    student = torch.randn(37, 90, generator=gen, device="cuda")
    values, indices = torch.topk(torch.randn(37, 90, generator=gen, device="cuda"), 5, dim=1)
    run(student, values, indices, torch.rand(37, generator=gen, device="cuda"), c=1.0 / 37)
