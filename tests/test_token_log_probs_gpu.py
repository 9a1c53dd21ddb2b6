"""Log-probabilities of drawn tokens far below the best one, where a weight of 2^-30 steps is a coarse measure: those of the
logits (``log_probs_of_logits``) against 64 bits.

Bound: (l - max) / T in fp32 is off by three roundings, 2^-22 |(l - max) / T|; the kept sum by 2^-31 of the best's weight a
token, relative to at least the best's; its logarithm by 2^-21 more."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.token_sampling import TokenSampler  # noqa: E402
from tests.test_token_sampling_gpu import full, plain  # noqa: E402


def _check(logits, u, least=None, **filters):
    rows, vocab = logits.shape
    tokens, drawn = torch.empty(rows, dtype=torch.int32, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")
    own, of_draw = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    op = TokenSampler(rows, vocab)
    op.run(logits=logits, uniforms=u, tokens=tokens, log_probs=own, log_probs_of_logits=True, **filters)
    op.run(logits=logits, uniforms=u, tokens=drawn, log_probs=of_draw, **filters)
    settings = {**dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **filters}
    want, kept, total = plain(logits, u, *(full(settings[k], rows, torch.int32 if k == "top_k" else torch.float32)
                                           for k in ("temperature", "top_k", "top_p", "min_p")))
    assert torch.equal(tokens, want) and torch.equal(drawn, want)
    t = float(torch.tensor(settings["temperature"]))
    x = logits.double()
    z = (x - x.amax(1, keepdim=True)) / t if t > 0 else torch.where(x == x.amax(1, keepdim=True), 0.0, -math.inf)
    exact = z.gather(1, want.long()[:, None])[:, 0] - torch.where(kept > 0, z.exp(), 0.0).sum(1).log()
    if t == 0:
        exact = torch.zeros_like(exact)
    at = z.gather(1, want.long()[:, None])[:, 0].abs()
    bound = 2.0 ** -22 * at + (kept > 0).sum(1) * 2.0 ** -31 + 2.0 ** -21 * (1 + exact.abs())
    assert bool(((own.double() - exact).abs() <= bound).all()), (own, exact, bound)
    mine = kept.gather(1, want.long()[:, None])[:, 0].double()
    assert bool(((of_draw.double() - (mine / total.double()).log()).abs() <= 1e-5).all())  # the draw's own, as before
    if least is not None:
        assert bool((at >= least).all())
    return own, of_draw


# a warp a row; a CTA a row from a list of few and of many candidates, and from the whole row; clusters
SIZES = [(40, 5), (40, 32), (40, 300), (40, 1024), (40, 3000), (200, 20000), (2, 140000)]


@pytest.mark.parametrize("rows,vocab", SIZES)
def test_one_token_far_down(rows, vocab):
    """Token 0 is 14 to 20.7 below the best, the rest has no weight; a uniform of 0 draws it."""
    logits = torch.full((rows, vocab), -30.0, device="cuda")
    logits[:, 0] = -torch.linspace(14.0, 20.7, rows, device="cuda")
    logits[:, vocab - 1] = 0.0
    u = torch.zeros(rows, device="cuda")
    worst = 0.0
    for filters in (dict(), dict(top_k=3), dict(top_k=vocab - 1), dict(temperature=1.0, min_p=1e-10)):
        own, of_draw = _check(logits, u, least=14.0, **filters)
        worst = max(worst, (own - of_draw).abs().max().item())
    assert worst > 1e-3  # the draw's are as coarse as they are said to be
    _check(logits * 0.7, u, least=13.9, temperature=0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [s for s in SIZES if s[1] >= 1024])
def test_many_tokens_far_down(rows, vocab, dtype):
    """700 tokens 12 to 20 below the best, drawn by uniforms that fall among them."""
    gen = torch.Generator(device="cuda").manual_seed(0)
    logits = torch.full((rows, vocab), -40.0, device="cuda")
    logits[:, :700] = -12.0 - 8.0 * torch.rand(rows, 700, generator=gen, device="cuda")
    logits[:, 900] = 0.0
    logits = logits.to(dtype)
    e = logits[:, :700].double().exp().sum(1)
    u = (torch.rand(rows, generator=gen, device="cuda") * 0.9 * (e / (1 + e))).float()
    for filters in (dict(), dict(top_k=800), dict(top_k=701), dict(min_p=1e-9)):
        _check(logits, u, least=11.9, **filters)


def test_ordinary_rows_and_the_best_token():
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(300, 500, generator=gen, device="cuda") * 3
    u = torch.rand(300, generator=gen, device="cuda")
    for filters in (dict(), dict(top_k=5), dict(top_p=0.7), dict(temperature=0.6, top_p=0.9, min_p=0.01), dict(temperature=0.0), dict(top_k=1)):
        _check(logits, u, **filters)
    logits[:, 3] = 60.0  # nothing but the best: 0, not a rounding of it
    own, _ = _check(logits, u)
    assert not bool(own.any())
    logits[7] = -math.inf
    tokens, lp = torch.empty(300, dtype=torch.int32, device="cuda"), torch.empty(300, device="cuda")
    TokenSampler(300, 500).run(logits=logits, uniforms=u, tokens=tokens, log_probs=lp, log_probs_of_logits=True)
    assert tokens[7] == -1 and lp[7] == -math.inf
