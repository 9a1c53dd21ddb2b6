"""Distillation of rows whose logits are large finite numbers: masks that fill a whole row with one, logits with a common
offset. A softmax does not see the offset, so loss and gradient are those of the differences."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.distillation import TopKDistillation  # noqa: E402
from tests.test_distillation_gpu import U, close, reference, run  # noqa: E402

# scaled by log2(e) / T these lie below, about and far above 2^24, 2^31 and 2^100
OFFSETS = [1.1e7, -1.1e7, 1.17e7, -1.17e7, 2.4e7, 3e8, -1e9, 3e9, -1e10, 1e20, -1e30, 2e38, -3e38]
SIZES = [(6, 70), (6, 700), (6, 2000), (6, 2500), (310, 2500), (6, 40000), (1, 300000)]


def _entries(rows, vocab, top, dtype):
    """A teacher on every third token from the end on."""
    indices = (vocab - 1 - 3 * torch.arange(top, device="cuda")).expand(rows, top).contiguous()
    gen = torch.Generator(device="cuda").manual_seed(1)
    return torch.randn(rows, top, generator=gen, device="cuda").to(dtype), indices, torch.rand(rows, generator=gen, device="cuda") + 0.5


def _held(want):
    """What fp32 makes of a value: infinity where it is larger than it holds (losses grow with T^2)."""
    return torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_rows_of_one_value(rows, vocab, dtype):
    """Every logit of the row the same: uniform, whatever the value."""
    values, indices, weight = _entries(rows, vocab, 8, dtype)
    for offset in OFFSETS:
        if abs(offset) > torch.finfo(dtype).max:
            offset = math.copysign(torch.finfo(dtype).max, offset)
        student = torch.full((rows, vocab), offset, dtype=dtype, device="cuda")
        for temperature in (1.0, 0.5, 0.001):
            row_loss, _, ds = run(student, values, indices, weight, temperature=temperature)
            assert bool(torch.isfinite(row_loss).all()) and bool(torch.isfinite(ds).all())


@pytest.mark.parametrize("rows,vocab", SIZES)
def test_differences_at_an_offset(rows, vocab):
    """fp32 logits of an offset and 0 to 40 steps of its last place, taken together with a temperature of a step: (max - s) / T
    is 0 to 40 as for ordinary logits."""
    values, indices, weight = _entries(rows, vocab, 8, torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(2)
    steps = torch.randint(0, 41, (rows, vocab), generator=gen, device="cuda")
    for offset in (1.1e7, -1.1e7, 2.4e7, 3e8, -1e9, 3e9, -1e10, 1e20, -1e25):
        step = 2.0 ** (math.frexp(abs(offset))[1] - 23)  # one step of the last place, or two
        student = (torch.tensor(offset).double().item() // step * step - steps.double() * step).float()
        assert bool((student.double() + steps.double() * step == student.double()[:, :1] + steps.double()[:, :1] * step).all())
        row_loss, loss, ds = torch.empty(rows, device="cuda"), torch.empty(1, device="cuda"), torch.empty(rows, vocab, device="cuda")
        TopKDistillation(rows, vocab, 8).run(logits=student, teacher_values=values, teacher_indices=indices, temperature=step,
                                             row_weight=weight, loss_weight=0.25, row_loss=row_loss, loss_out=loss, dlogits=ds)
        of_row, of_all, grad = reference(student, values, indices, step, weight, 0.25, 1.0)
        close("row_loss", row_loss, _held(of_row[0]), of_row[1])
        close("loss", loss[0], _held(of_all[0]), of_all[1])
        close("dlogits", ds, grad[0], grad[1] + U[torch.float32] * grad[0].abs() + 2.0 ** -126)


@pytest.mark.parametrize("rows,vocab", SIZES)
def test_masked_rows_beside_ordinary_ones(rows, vocab):
    """-1e10 in the masked places of some rows, in all places of others."""
    values, indices, weight = _entries(rows, vocab, 8, torch.float32)
    gen = torch.Generator(device="cuda").manual_seed(3)
    student = torch.randn(rows, vocab, generator=gen, device="cuda") * 3
    masked = torch.rand(rows, vocab, generator=gen, device="cuda") < 0.5
    masked.scatter_(1, indices, False)
    masked[::2] = True
    run(student.masked_fill(masked, -1e10), values, indices, weight, temperature=2.0)
