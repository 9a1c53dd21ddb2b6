"""The token policy: logits, loss and gradients of the fp16 recipe against the same network in 64 bits
(1e-2, the fp16 recipe's tolerance of this suite), learning, acting, and a CUDA graph of a whole step."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.token_policy import TokenPolicy  # noqa: E402


def _teacher(rows, tokens, top, gen):
    values, indices = torch.topk(torch.randn(rows, tokens, generator=gen, device="cuda") * 2, top, dim=1)
    return values, indices


def _reference(policy, obs, values, indices, temperature):
    """Loss and gradients by autograd in 64 bits from the fp16 weight planes and fp16 observations."""
    w = {k: v.plane(policy.planes).double().requires_grad_() for k, v in policy.weights.items()}
    x = obs.half().double()
    h0 = x @ w["in"].t()
    h1 = h0 + (torch.nn.functional.silu(h0 @ w["gate"].t()) * (h0 @ w["up"].t())) @ w["down"].t()
    logits = h1 @ w["head"].t()
    q = torch.softmax(values.double() / temperature, 1)
    log_p = torch.log_softmax(logits / temperature, 1).gather(1, indices)
    loss = temperature ** 2 * (q * (q.log() - log_p)).sum(1).mean()
    loss.backward()
    return logits, loss, {k: v.grad for k, v in w.items()}


@pytest.mark.parametrize("obs_dim,tokens,rows,hidden,temperature", [(31, 101, 300, 64, 1.0), (40, 3000, 128, 96, 2.0)])
def test_step_against_autograd(obs_dim, tokens, rows, hidden, temperature):
    gen = torch.Generator(device="cuda").manual_seed(0)
    policy = TokenPolicy(obs_dim, tokens, rows, hidden=hidden, top=7)
    obs = torch.randn(rows, obs_dim, generator=gen, device="cuda")
    values, indices = _teacher(rows, tokens, 7, gen)
    logits, loss, grads = _reference(policy, obs, values, indices, temperature)
    policy.load_observations(obs)
    policy.gradients(values, indices, temperature)
    close = lambda a, b: float((a.detach().double() - b.detach()).norm() / b.detach().norm())  # noqa: E731
    assert close(policy.logits[:, :tokens], logits) < 1e-2
    assert abs(policy.loss.item() - float(loss.detach())) < 1e-2 * float(loss.detach())
    for name, w in policy.weights.items():
        assert close(w.arena(policy.grads), grads[name]) < 1e-2, name
    assert policy.health.item() == 0 and policy.found_inf.item() == 0


def test_learns_and_acts():
    rows, obs_dim, tokens, top = 512, 32, 64, 8
    gen = torch.Generator(device="cuda").manual_seed(1)
    teacher = TokenPolicy(obs_dim, tokens, rows, hidden=64, seed=5)
    student = TokenPolicy(obs_dim, tokens, rows, hidden=64, seed=6, top=top, learning_rate=2e-3)
    losses = []
    for _ in range(150):
        obs = torch.randn(rows, obs_dim, generator=gen, device="cuda")
        teacher.load_observations(obs)
        values, indices = torch.topk(teacher.forward() * 2.0, top, dim=1)
        losses.append(student.distill_update(obs, values, indices).item())
    assert losses[-1] < 0.6 * losses[0]
    tokens_drawn, log_probs = student.act(obs, torch.rand(rows, generator=gen, device="cuda"), top_k=1)
    assert torch.equal(tokens_drawn.long(), student.logits[:, :tokens].argmax(1)) and not bool(log_probs.any())
    assert student.health.item() == 0


def test_step_in_a_graph():
    gen = torch.Generator(device="cuda").manual_seed(2)
    obs = torch.randn(64, 20, generator=gen, device="cuda")
    values, indices = _teacher(64, 50, 4, gen)
    eager, graphed = (TokenPolicy(20, 50, 64, hidden=32, top=4, seed=3) for _ in range(2))
    eager.distill_update(obs, values, indices)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        graphed.distill_update(obs, values, indices)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager.params, graphed.params) and torch.equal(eager.loss, graphed.loss)
