"""Token sampling (``rl2_sample_tokens``): bit for bit against the definition with integer weights, and
against the probabilities in 64 bits."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.token_sampling import TokenSampler  # noqa: E402

INF = math.inf


def plain(logits, u, temperature, top_k, top_p, min_p):
    """The definition on [rows, vocab] logits; the parameters are [rows] tensors. Also the kept weights."""
    x = logits.float()
    x = torch.where(torch.isnan(x), -INF, x).clamp(max=torch.finfo(torch.float32).max)
    V = x.shape[1]
    best = x.amax(1, keepdim=True)
    empty = best == -INF
    t = temperature.float()[:, None]
    e = torch.exp((x - best) * (torch.ones_like(t) / t))
    w = torch.where(torch.isnan(e), 0.0, torch.round(e * 2.0 ** 30)).long()
    greedy = t == 0
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    rank = torch.arange(V, device=x.device)[None]
    ranked = w.gather(1, order)
    k = top_k[:, None]
    ranked = torch.where((k > 0) & (rank >= k), 0, ranked)
    before = ranked.cumsum(1) - ranked
    p = top_p.float().double()[:, None]
    keep = (p >= 1) | (before.double() < p * ranked.sum(1, keepdim=True).double()) & (p > 0) | (rank == 0)
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, ranked, 0))
    kept = torch.where(e >= min_p.float()[:, None], kept, 0)
    first = torch.zeros_like(w).scatter_(1, order, (rank == 0).long().expand_as(w).contiguous())
    kept = torch.where(greedy, first, kept)
    total = kept.sum(1, keepdim=True)
    at = torch.where(u >= 0, u, 0).double()[:, None] * total.double()
    target = torch.minimum(at.long(), total - 1)
    token = (kept.cumsum(1) > target).int().argmax(1)
    return torch.where(empty[:, 0], -1, token).int(), kept, total[:, 0]


def full(value, rows, dtype=torch.float32):
    return value if isinstance(value, torch.Tensor) else torch.full((rows,), value, dtype=dtype, device="cuda")


def check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, op=None):
    R, V = logits.shape
    op = op or TokenSampler(max(R, 1), V)
    tokens = torch.full((R,), -7, dtype=torch.int32, device="cuda")
    lp = torch.full((R,), math.nan, device="cuda")
    op.run(logits=logits, uniforms=u, tokens=tokens, log_probs=lp, temperature=temperature, top_k=top_k, top_p=top_p,
           min_p=min_p)
    want, kept, total = plain(logits, u, full(temperature, R), full(top_k, R, torch.int32), full(top_p, R), full(min_p, R))
    assert torch.equal(tokens, want), (tokens[tokens != want][:5], want[tokens != want][:5])
    mine = kept.gather(1, want.clamp(min=0).long()[:, None])[:, 0].double()
    exact = torch.where(want < 0, -INF, (mine / total.double()).log())
    # 1 fp32 rounding each of w, W, their quotient and the logarithm (2 units): 4 * 2^-23 relative to 1 + |log|
    ok = (lp == exact) | ((lp - exact).abs() <= 5e-7 * (exact.abs() + (exact.abs() > 0.6)))
    assert bool(ok.all()), (lp[~ok][:5], exact[~ok][:5])
    return tokens, lp


def draws(rows, vocab, dtype=torch.float32, seed=0, scale=3.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=gen, device="cuda") * scale).to(dtype)
    return logits, torch.rand(rows, generator=gen, device="cuda")


FILTERS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=1), dict(top_k=5), dict(top_p=0.3), dict(top_p=0.0),
           dict(temperature=1.7, top_p=0.95), dict(min_p=0.05), dict(min_p=1.0), dict(top_k=40, top_p=0.8, min_p=0.01, temperature=0.9)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(3, 1), (5, 2), (64, 31), (33, 32), (200, 101), (300, 256), (65, 1000), (40, 1024), (17, 1025), (20, 4096),
                                        (9, 4097), (13, 32000), (150, 5003), (3, 50257), (2, 128257), (1, 262144), (1, 1 << 20)])
def test_definition(rows, vocab, dtype):
    logits, u = draws(rows, vocab, dtype, seed=vocab)
    op = TokenSampler(rows, vocab)
    for f in FILTERS:
        check(logits, u, op=op, **f)


@pytest.mark.parametrize("vocab", [7, 256, 1024, 3000, 40000, 140001])
def test_parameters_of_each_row(vocab):
    rows = 48
    logits, u = draws(rows, vocab, torch.bfloat16, seed=5)
    gen = torch.Generator(device="cuda").manual_seed(6)
    t = torch.rand(rows, generator=gen, device="cuda") * 2
    t[::7] = 0
    k = torch.randint(-1, vocab + 2, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    p = torch.rand(rows, generator=gen, device="cuda") * 1.2
    m = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.5, 0.0, torch.rand(rows, generator=gen, device="cuda"))
    check(logits, u, t, k, p, m)


@pytest.mark.parametrize("vocab", [6, 300, 1024, 9000, 140000])
def test_ties_fall_to_the_lowest_index(vocab):
    """Few different values: every cut falls inside a run of equal logits; and all logits equal."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randint(0, 4, (24, vocab), generator=gen, device="cuda").float()
    logits[:6] = 2.5
    logits[6:12].mul_(-0.0)  # both zeros are one value
    u = torch.rand(24, generator=gen, device="cuda")
    for f in (dict(top_k=3), dict(top_p=0.37), dict(top_k=vocab // 2 + 1, top_p=0.61), dict(temperature=0.0), dict(top_k=vocab - 1)):
        check(logits, u, **f)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [16, 513, 1024, 20000, 140000])
def test_masks(vocab, dtype):
    logits, u = draws(12, vocab, dtype, seed=2)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits[0] = -INF
    logits[1] = math.nan
    logits[2] = low
    logits[3, 1:] = -INF
    logits[4, :-1] = low
    logits[5, vocab // 2] = INF
    logits[6, ::3] = math.nan
    logits[7, ::2] = -INF
    logits[8, :3] = INF
    logits[9] = high
    logits[10, : vocab - 1] = -INF
    for f in FILTERS:
        tokens, _ = check(logits, u, **f)
        assert tokens[0] == -1 and tokens[1] == -1 and tokens[3] == 0 and tokens[10] == vocab - 1


@pytest.mark.parametrize("rows,vocab", [(5, 300), (3, 6000), (200, 20000), (2, 140000)])
def test_temperatures_at_the_ends(rows, vocab):
    """So low that only the best count, so high that all weigh the same, and what is no normal number."""
    logits, u = draws(rows, vocab, seed=vocab)
    for t in (1e-45, 1e-38, 1.5e-38, 1e-36, 1e-30, 1e-4, 1e4, 1e30, INF):
        gone = dict(temperature=0.0) if t < 2.0 ** -126 else dict(temperature=t)
        tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
        for f in (dict(), dict(top_k=7), dict(top_p=0.5), dict(top_k=min(vocab, 900), top_p=0.9), dict(min_p=0.5)):
            want, _ = check(logits, u, **gone, **f)
            TokenSampler(rows, vocab).run(logits=logits, uniforms=u, tokens=tokens, temperature=t, **f)
            assert torch.equal(tokens, want)


@pytest.mark.parametrize("rows,vocab,spread", [(2, 20000, 1e-4), (200, 9000, 1e-3), (2, 200000, 1e-38), (100, 70000, 0.5), (1, 50000, 100.0)])
def test_narrow_and_wide_rows(rows, vocab, spread):
    """All tokens near one another (one histogram bin holds more than a list), and very far."""
    logits, u = draws(rows, vocab, seed=3, scale=spread)
    for f in (dict(), dict(top_k=vocab // 3), dict(top_p=0.5), dict(top_k=5000, top_p=0.3), dict(top_k=100, top_p=0.999), dict(min_p=0.9)):
        check(logits, u, **f)


@pytest.mark.parametrize("vocab", [5, 777, 33333, 150000])
def test_probabilities_in_64_bits(vocab):
    """The drawn token's interval of the cumulative probabilities, in 64 bits from the definition, holds the
    uniform to within the error of fp32 exponentials and of weights rounded to 2^-30."""
    rows = 40
    logits, u = draws(rows, vocab, seed=11)
    op = TokenSampler(rows, vocab)
    tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
    op.run(logits=logits, uniforms=u, tokens=tokens, temperature=0.8, top_k=50)
    x = logits.double()
    e = torch.exp((x - x.amax(1, keepdim=True)) / torch.tensor(0.8).double())
    if vocab > 50:
        e = torch.where(x >= torch.topk(x, 50, dim=1).values[:, -1:], e, 0.0)
    cdf = e.cumsum(1) / e.sum(1, keepdim=True)
    upper = cdf.gather(1, tokens.long()[:, None])[:, 0]
    share = (e / e.sum(1, keepdim=True)).gather(1, tokens.long()[:, None])[:, 0]
    slack = 2.0 ** -22 * 30 + 50 * 2.0 ** -30  # relative error of e: 2 units + (l - max) / T rounded, |.| < 30
    assert bool((share > 0).all())
    assert bool((u.double() <= upper + slack).all()) and bool((u.double() >= upper - share - slack).all())


def test_uniforms_at_the_ends():
    logits, _ = draws(5, 300)
    u = torch.tensor([0.0, -1.0, math.nan, 1.0, 2.0], device="cuda")
    tokens, _ = check(logits, u)
    assert tokens[:3].tolist() == [0, 0, 0] and tokens[3:].tolist() == [299, 299]


@pytest.mark.parametrize("vocab", [100, 5000, 70001])
def test_rows_of_a_wider_matrix(vocab):
    """Strides and alignments: views of a wider matrix, poisoned beside them, on another stream."""
    wide, u = draws(9, vocab + 13, torch.bfloat16)
    for first in (0, 1, 3, 8):
        view = wide[:, first:first + vocab]
        want, _ = check(view.contiguous(), u, top_k=20)
        poisoned = torch.full_like(wide, INF)
        poisoned[:, first:first + vocab] = view
        tokens = torch.empty(9, dtype=torch.int32, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        TokenSampler(9, vocab).run(logits=poisoned[:, first:first + vocab], uniforms=u, tokens=tokens, top_k=20, stream=side)
        side.synchronize()
        assert torch.equal(tokens, want)


def test_many_rows_no_rows_and_graph():
    logits, u = draws(5000, 64)
    check(logits, u, top_p=0.9)
    op = TokenSampler(4, 9000)
    empty = torch.empty(0, 9000, device="cuda")
    op.run(logits=empty, uniforms=empty[:, 0], tokens=torch.empty(0, dtype=torch.int32, device="cuda"))
    logits, u = draws(4, 9000)
    want, _ = check(logits, u, top_k=10, top_p=0.9)
    tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run(logits=logits, uniforms=u, tokens=tokens, top_k=10, top_p=0.9)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(tokens, want)


def test_rows_with_parameters_out_of_range():
    logits, u = draws(4, 50)
    op = TokenSampler(4, 50)
    tokens = torch.zeros(4, dtype=torch.int32, device="cuda")
    for name, bad in (("temperature", -1.0), ("temperature", math.nan), ("top_p", math.nan), ("min_p", 1.5)):
        health = torch.zeros(1, dtype=torch.int32, device="cuda")
        value = torch.full((4,), 0.5, device="cuda")
        value[2] = bad
        op.run(logits=logits, uniforms=u, tokens=tokens, health=health, **{name: value})
        assert tokens[2] == -1 and bool((tokens[[0, 1, 3]] >= 0).all()) and health.item() == 8


def test_refusals():
    for rows, vocab in ((0, 5), (5, 0), (5, (1 << 20) + 1)):
        with pytest.raises(ValueError, match="rows must be"):
            TokenSampler(rows, vocab)
    op = TokenSampler(4, 50)
    logits, u = draws(4, 50)
    good = dict(logits=logits, uniforms=u, tokens=torch.zeros(4, dtype=torch.int32, device="cuda"))

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            op.run(**{**good, **change})

    refused(ValueError, "logits must be", logits=logits.double())
    refused(ValueError, "logits must be", logits=logits[:, :49])
    refused(ValueError, "logits must be", logits=logits.cpu())
    refused(ValueError, "contiguous rows", logits=torch.zeros(50, 4, device="cuda").t())
    refused(ValueError, "uniforms must be", uniforms=u[:3])
    refused(ValueError, "tokens must be", tokens=good["tokens"].long())
    refused(ValueError, "log_probs must be", log_probs=u.half())
    refused(ValueError, "top_k must be", top_k=u)
    refused(RuntimeError, "temperature >= 0", temperature=-0.1)
    refused(RuntimeError, "temperature >= 0", temperature=math.nan)
    refused(RuntimeError, "min_p <= 1", min_p=1.1)
    refused(RuntimeError, "shorter than a row", logits=logits[:1].expand(4, 50))
