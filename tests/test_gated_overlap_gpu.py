"""The gated block refuses outputs that share memory with what is still read: nothing is launched. Views side by side in
one buffer, a gradient in place of grad_out, a weight's in place of the weight are no such case, and give the same bits."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.gated import GatedMLP  # noqa: E402


def _operands(rows, width):
    gen = torch.Generator(device="cuda").manual_seed(0)
    return [(torch.randn(n, width, generator=gen, device="cuda") * 0.1).half() for n in (rows, width, width, rows)]


@pytest.mark.parametrize("rows", [2, 40, 200])
def test_forward(rows):
    width = 64
    x, wg, wu, _ = _operands(rows, width)
    op = GatedMLP(rows, width, width)
    room = torch.zeros(rows + 4, 2 * width, dtype=torch.float16, device="cuda")
    room[:rows, :width] = x
    inside = room[:rows, :width]
    for out in (inside, room[1:rows + 1, :width], room[:rows, 8:width + 8], room.view(-1)[:rows * width].view(rows, width)):
        with pytest.raises(RuntimeError, match="may not overlap"):
            op.forward(x=inside, gate_weight=wg, up_weight=wu, out=out)
    big = torch.zeros(2 * width, width, dtype=torch.float16, device="cuda")
    big[:width] = wg
    if rows <= width:
        with pytest.raises(RuntimeError, match="may not overlap"):
            op.forward(x=x, gate_weight=big[:width], up_weight=wu, out=big[width - 1:width - 1 + rows])
    assert torch.equal(inside, x) and torch.equal(big[:width], wg)
    want = torch.empty_like(x)
    op.forward(x=x, gate_weight=wg, up_weight=wu, out=want)
    op.forward(x=inside, gate_weight=wg, up_weight=wu, out=room[:rows, width:])  # beside it
    assert torch.equal(room[:rows, width:], want) and torch.equal(inside, x)


@pytest.mark.parametrize("rows", [2, 200])
def test_backward(rows):
    width = 64
    x, wg, wu, dh = _operands(rows, width)
    op = GatedMLP(rows, width, width)
    make = lambda n: torch.empty(n, width, dtype=torch.float16, device="cuda")  # noqa: E731
    dx, dg, du = make(rows), make(width), make(width)
    good = dict(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx, grad_gate=dg, grad_up=du)
    op.backward(**good)
    room = torch.zeros(2 * rows + 2 * width, width, dtype=torch.float16, device="cuda")

    def refused(**change):
        with pytest.raises(RuntimeError, match="may not overlap"):
            op.backward(**{**good, **change})

    refused(x=room[:rows], grad_x=room[1:rows + 1])
    refused(gate_weight=room[:width], grad_x=room[width - 1:width - 1 + rows])
    refused(up_weight=room[:width], grad_x=room[width - 1:width - 1 + rows])
    refused(x=room[:rows], grad_gate=room[rows - 1:rows - 1 + width])
    refused(x=room[:rows], grad_up=room[rows - 1:rows - 1 + width])
    refused(grad_gate=room[:width], grad_up=room[width - 1:2 * width - 1])
    refused(grad_x=room[:rows], grad_gate=room[rows - 1:rows - 1 + width])
    assert not bool(room.any())
    # in place of what is done with: the same bits
    dh2, wg2, wu2 = dh.clone(), wg.clone(), wu.clone()
    op.backward(x=x, gate_weight=wg2, up_weight=wu2, grad_out=dh2, grad_x=dh2, grad_gate=wg2, grad_up=wu2)
    assert torch.equal(dh2, dx) and torch.equal(wg2, dg) and torch.equal(wu2, du)
    # without weight gradients x is not read again
    shifted = torch.cat([x, torch.zeros_like(x[:1])])
    op.backward(x=shifted[:rows], gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=shifted[1:])
    assert torch.equal(shifted[1:], dx)
