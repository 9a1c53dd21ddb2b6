"""GELU in its lower tail: g Phi(g) and its derivative keep their relative accuracy where 1 + erf has none left. x holds one
g per row and a 1, so that g, u and the gradients are single products.

Bounds, relative: the exponential of g^2 / 2 carries the rounding of its argument, 2 g^2 2^-24, and (2 + 1.17 g^2 / 2) units
of the function; Phi 5e-7 more; the derivative's two terms cancel to two thirds at most from g = -2 on. Then one rounding of
each output, and of dg and du before the last product."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.gated import GatedMLP  # noqa: E402

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ETA = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}  # bf16 results below the smallest normal number may be 0
UP = 512.0


def _formula(g):
    g = g.double()
    cdf = 0.5 * torch.special.erfc(-g / math.sqrt(2.0))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _rows(rows, dtype):
    """g from -13 to -2 (fp16: to where 512 g Phi(g) is a normal number), as the type holds it."""
    return torch.linspace(-13.0 if dtype == torch.bfloat16 else -6.5, -2.0, rows, device="cuda").to(dtype)


def _operands(rows, dtype):
    g = _rows(rows, dtype)
    x = torch.zeros(rows, 8, dtype=dtype, device="cuda")
    x[:, 0], x[:, 1] = g, 1.0
    wg, wu = (torch.zeros(16, 8, dtype=dtype, device="cuda") for _ in range(2))
    wg[:, 0], wu[:, 1] = 1.0, UP
    return g, x, wg, wu


def _fp32(g):
    g2 = g.double().square()
    return 5e-7 + 2 * g2 * 2.0 ** -24 + (2 + 0.6 * g2) * 2.0 ** -23


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 7, 16, 17, 100, 128, 129, 1000])
def test_value(rows, dtype):
    g, x, wg, wu = _operands(rows, dtype)
    h = torch.empty(rows, 16, dtype=dtype, device="cuda")
    GatedMLP(rows, 8, 16, dtype=dtype, activation="gelu").forward(x=x, gate_weight=wg, up_weight=wu, out=h)
    want = (_formula(g)[0] * UP)[:, None].expand(rows, 16)
    assert bool(((h.double() - want).abs() <= (U[dtype] + _fp32(g)[:, None]) * want.abs() + ETA[dtype]).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 40, 129, 1000])
def test_gradients(rows, dtype):
    """dh = 512 for one hidden unit: dx[:, 0] = dg, dx[:, 1] = 512 du."""
    g, x, wg, wu = _operands(rows, dtype)
    dh = torch.zeros(rows, 16, dtype=dtype, device="cuda")
    dh[:, 3] = UP
    dx = torch.empty_like(x)
    GatedMLP(rows, 8, 16, dtype=dtype, activation="gelu").backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx)
    value, slope = _formula(g)
    for column, want, hidden in ((0, slope * UP * UP, 1.0), (1, value * UP * UP, UP)):
        if not bool((want.abs() < torch.finfo(dtype).max).all()):
            want = want.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)
        bound = (2 * U[dtype] + 3 * _fp32(g)) * want.abs() + ETA[dtype] * (1 + hidden)
        assert bool(((dx[:, column].double() - want).abs() <= bound).all()), column


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_whole_range(dtype):
    """And everywhere else: values between -4 and 8, dx and h to their absolute size."""
    rows = 4000
    g = torch.linspace(-4.0, 8.0, rows, device="cuda").to(dtype)
    _, x, wg, wu = _operands(rows, dtype)
    x[:, 0], wu[:, 1] = g, 1.0
    h, dx, dh = torch.empty(rows, 16, dtype=dtype, device="cuda"), torch.empty_like(x), torch.zeros(rows, 16, dtype=dtype, device="cuda")
    dh[:, 3] = 1.0
    op = GatedMLP(rows, 8, 16, dtype=dtype, activation="gelu")
    op.forward(x=x, gate_weight=wg, up_weight=wu, out=h)
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx)
    value, slope = _formula(g)
    for got, want, roundings in ((h[:, 5], value, 1), (dx[:, 1], value, 2), (dx[:, 0], slope, 2)):
        assert bool(((got.double() - want).abs() <= roundings * U[dtype] * want.abs() + 2 * ETA[dtype] + 1e-6 * (1 + g.double().abs())).all())
