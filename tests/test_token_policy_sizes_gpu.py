"""The token policy at sizes that fill no whole 16 bytes: hidden and expanded widths of any remainder."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.token_policy import TokenPolicy  # noqa: E402
from tests.test_token_policy_gpu import _reference, _teacher  # noqa: E402


@pytest.mark.parametrize("obs_dim,tokens,rows,hidden,expand", [(24, 50, 64, 100, 1), (24, 50, 64, 50, 4), (7, 13, 5, 33, 3), (31, 101, 300, 61, 2),
                                                               (8, 9, 140, 99, 1), (3, 5, 20, 6, 3)])
def test_step_against_autograd(obs_dim, tokens, rows, hidden, expand):
    """1e-2: the fp16 recipe's tolerance of this suite."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    policy = TokenPolicy(obs_dim, tokens, rows, hidden=hidden, expand=expand, top=4)
    obs = torch.randn(rows, obs_dim, generator=gen, device="cuda")
    values, indices = _teacher(rows, tokens, 4, gen)
    logits, loss, grads = _reference(policy, obs, values, indices, 1.0)
    before = {name: w.arena(policy.params).clone() for name, w in policy.weights.items()}
    assert torch.equal(policy.distill_update(obs, values, indices), policy.loss)
    close = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())  # noqa: E731
    assert close(policy.logits[:, :tokens], logits) < 1e-2
    assert abs(policy.loss.item() - float(loss.detach())) < 1e-2 * float(loss.detach())
    for name, w in policy.weights.items():
        assert close(w.arena(policy.grads), grads[name]) < 1e-2, name
        moved = (w.arena(policy.params) - before[name]).abs()
        assert moved.max().item() <= 3.1e-4 and bool((moved > 0).float().mean() > 0.5)  # Adam's first step: the learning rate each
        assert torch.equal(w.plane(policy.planes), w.arena(policy.params).half())
    assert policy.health.item() == 0 and policy.found_inf.item() == 0
    tokens_drawn, _ = policy.act(obs, torch.rand(rows, generator=gen, device="cuda"), top_k=1)
    assert torch.equal(tokens_drawn.long(), policy.logits[:, :tokens].argmax(1))
