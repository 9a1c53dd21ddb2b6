"""Overflow inside the gated block's backward (``found_inf`` of ``rl2_gated_backward``): hidden gradients and outputs
that their type does not hold are reported, and the token policy's optimizer skips such a step. All operands are chosen so
that every value is known: one feature of x is 1, the others 0, ReLU with g > 0, so g and u are columns of the weights."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.gated import GatedMLP  # noqa: E402
from robolearn_b200.token_policy import TokenPolicy  # noqa: E402

LARGEST = {torch.float16: 65504.0, torch.bfloat16: 3.3895313892515355e38}


def _run(rows, features, hidden, dtype, gate, up, dh, *, weights=None, with_x=True, report=True, flag=0, at=None):
    """found_inf and health after a backward pass whose g, u and dh are constants, or only in hidden unit ``at`` (elsewhere 1)."""
    def plane(r, c, value):
        t = torch.zeros(r, (c + 7) // 8 * 8, dtype=dtype, device="cuda")[:, :c]
        return t.copy_(value) if isinstance(value, torch.Tensor) else t.fill_(value)

    def column(value):
        t = torch.zeros(hidden, features, device="cuda")
        t[:, 0] = value if at is None else 1.0
        if at is not None:
            t[at, 0] = value
        return t

    x = torch.zeros(rows, features, device="cuda")
    x[:, 0] = 1.0
    x, wg, wu, dh = plane(rows, features, x), plane(hidden, features, column(gate)), plane(hidden, features, column(up)), plane(rows, hidden, dh)
    found = torch.full((1,), flag, dtype=torch.int32, device="cuda")
    health = torch.zeros(1, dtype=torch.int32, device="cuda")
    dx = plane(rows, features, 0.0) if with_x else None
    dw = (None, None)
    if weights is not None:
        ld = (features + 7) // 8 * 8
        dw = tuple(torch.zeros(hidden, ld, dtype=weights, device="cuda")[:, :features] for _ in range(2))
    op = GatedMLP(rows, features, hidden, dtype=dtype, activation="relu")
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx, grad_gate=dw[0], grad_up=dw[1],
                found_inf=found if report else None, health=health)
    return found.item(), health.item()


# few rows, ragged tiles, several tiles; the contraction over the hidden units split (40 x 200 x 5000), over the rows (17000)
SIZES = [(1, 16, 40), (3, 24, 200), (130, 40, 333), (300, 64, 512), (40, 200, 5000), (17000, 24, 128)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,features,hidden", SIZES)
def test_hidden_gradients(rows, features, hidden, dtype):
    """dg = dh u and du = dh g of a single hidden unit, one past the largest value; dx then adds up from infinities."""
    root = LARGEST[dtype] ** 0.5
    for unit in (0, hidden // 2, hidden - 1):
        for gate, up in ((1.0, 2 * root), (2 * root, 1.0)):
            assert _run(rows, features, hidden, dtype, gate, up, root, at=unit) == (1, 0)
    if hidden * 4 * rows < 60000:  # and what fits is not reported (dx adds up hidden units, fp32 dW rows)
        assert _run(rows, features, hidden, dtype, 1.0, 1.0, 2.0, weights=torch.float32) == (0, 0)
        assert _run(rows, features, hidden, dtype, 1.0, 1.0, 2.0, weights=dtype) == (0, 0)


@pytest.mark.parametrize("rows,features,hidden", SIZES)
def test_input_gradient(rows, features, hidden):
    """dg and du fit, their sum over the hidden units (dx = 2 hidden dh) does not: reported by the call that writes dx alone."""
    assert _run(rows, features, hidden, torch.float16, 1.0, 1.0, 65504.0 / hidden * 0.75) == (1, 0)
    assert _run(rows, features, hidden, torch.float16, 1.0, 1.0, 65504.0 / hidden * 0.75, weights=torch.float32, with_x=False) == (0, 0)
    assert _run(rows, features, hidden, torch.float16, 1.0, 1.0, 65504.0 / hidden * 0.25) == (0, 0)


@pytest.mark.parametrize("rows,features,hidden", [s for s in SIZES if s[0] > 100])
def test_weight_gradients(rows, features, hidden):
    """A sum over the rows that fp16 does not hold and fp32 does."""
    dh = 65504.0 / rows * 1.5
    assert _run(rows, features, hidden, torch.float16, 1.0, 1.0, dh, weights=torch.float16, with_x=False) == (1, 0)
    assert _run(rows, features, hidden, torch.float16, 1.0, 1.0, dh, weights=torch.float32, with_x=False) == (0, 0)
    assert _run(rows, features, hidden, torch.float16, 1.0, 1.0, dh / 2, weights=torch.float16, with_x=False) == (0, 0)


@pytest.mark.parametrize("rows,hidden", [(3, 200), (300, 512)])
def test_largest_value_not_a_number_and_flags(rows, hidden):
    size = (rows, 24, hidden, torch.float16)
    assert _run(*size, 1.0, 65504.0, 1.0, at=7, weights=torch.float32, with_x=False) == (0, 0)  # dg is the largest value itself
    assert _run(*size, 1.0, 1.0, float("nan"), weights=torch.float32) == (1, 0)
    assert _run(*size, 1.0, 1.0, float("inf"), weights=torch.float32, with_x=False) == (1, 0)
    assert _run(*size, 1.0, 1.0, 1.0, flag=1) == (1, 0)  # what an earlier part of the step found stays
    assert _run(*size, 1.0, 1000.0, 1000.0, report=False) == (0, 4)  # without a flag: the health word's overflow bit
    assert _run(*size, 1.0, 1.0, 1.0, report=False) == (0, 0)


def test_flag_is_checked():
    with pytest.raises(ValueError, match="found_inf must be"):
        x, w, h = (torch.zeros(n, 16, dtype=torch.float16, device="cuda") for n in (4, 16, 4))
        GatedMLP(4, 16, 16).backward(x=x, gate_weight=w, up_weight=w, grad_out=h, grad_x=h.clone(), found_inf=torch.zeros(1, device="cuda"))


@pytest.mark.parametrize("rows", [48, 600])
def test_step_with_an_overflow_in_the_block_is_skipped(rows):
    """Up projections a thousand times their size: the gradients that reach the block are finite, dg is not."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    policy = TokenPolicy(24, 50, rows, hidden=64, top=4)
    policy.weights["up"].arena(policy.params).mul_(1000.0)
    policy.refresh_planes()
    obs = torch.randn(rows, 24, generator=gen, device="cuda")
    values, indices = torch.topk(torch.randn(rows, 50, generator=gen, device="cuda") * 2, 4, dim=1)
    policy.scale.fill_(2.0 ** 24)
    policy.inverse_scale.fill_(2.0 ** -24)
    policy.opt_state[6] = 2.0 ** 24
    for _ in range(24):  # the dynamic scale comes down until the gradients that reach the block fit
        policy.load_observations(obs)
        policy.gradients(values, indices)
        if bool(torch.isfinite(policy._dgated).all()) and bool(torch.isfinite(policy._dh1).all()):
            break
        policy._optimizer()
    assert policy.found_inf.item() == 1 and not bool(torch.isfinite(policy.grads).all())
    before = [t.clone() for t in (policy.params, policy.m1, policy.m2, policy.planes, policy.scale)]
    policy._optimizer()
    for t, old in zip((policy.params, policy.m1, policy.m2, policy.planes), before):
        assert torch.equal(t, old)
    assert policy.scale.item() == before[4].item() / 2 and policy.found_inf.item() == 0
    for _ in range(40):  # and it goes on: scales at which everything fits are found, the parameters stay numbers
        policy.distill_update(obs, values, indices)
    assert bool(torch.isfinite(policy.params).all()) and policy.opt_state[1].item() >= 1 and policy.health.item() == 0
