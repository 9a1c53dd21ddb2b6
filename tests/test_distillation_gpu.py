"""Distillation from a teacher's top logits (``rl2_distill_topk``) against the formulas in 64 bits.

Bounds: an exponential exp2((s - max) c) carries 2 units of the special function plus the rounded
argument, 2^-22 (1 + z) relative at z = (max - s) / T; a sum of n such terms adds (n / 32 + 40) 2^-24
(per-lane partial sums, then a tree), and the mean of z under softmax is at most ln n."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.distillation import TopKDistillation  # noqa: E402

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ETA = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
INF = math.inf


def reference(logits, values, indices, temperature, weight, c, grad_scale):
    """row_loss, loss, gradient and their bounds (without the gradient's own rounding)."""
    t = float(torch.tensor(temperature))
    s, v = logits.double() / t, values.double() / t
    N, V = s.shape
    K = v.shape[1]
    here = (indices >= 0) & (indices < V)
    at = torch.where(here, indices, 0).long()
    v = torch.where(here, v, -INF)
    top, best = v.amax(1, keepdim=True), s.amax(1, keepdim=True)
    some = ((top > -INF) & (best > -INF))[:, 0] & (weight != 0)
    zq, zs = torch.where(some[:, None], top - v, INF), torch.where(some[:, None], best - s, INF)
    q, p = torch.exp(-zq), torch.exp(-zs)
    q, p = q / q.sum(1, keepdim=True), p / p.sum(1, keepdim=True)
    q, p = torch.where(some[:, None], q, 0.0), torch.where(some[:, None], p, 0.0)
    unit = 2.0 ** -22
    err_sum = unit * (2 + math.log(V)) + (V / 32 + 40) * 2.0 ** -24
    err_q = unit * (3 + math.log(K)) + (K / 32 + 40) * 2.0 ** -24
    log_q, log_p = torch.log(q.clamp(min=1e-300)), torch.log(p).gather(1, at)
    term = torch.where(q > 0, q * (log_q - log_p), 0.0)
    row_loss = t * t * term.sum(1)
    size = torch.where(q > 0, q * (log_q.abs() + log_p.abs()), 0.0)
    grow = err_q + unit * torch.nan_to_num(zq, posinf=0.0)
    row_bound = t * t * torch.where(q > 0, size * (grow + unit + (K / 32 + 40) * 2.0 ** -24) + q * (err_q + err_sum + 2 * unit), 0.0).sum(1)
    scattered = torch.zeros_like(p).scatter_add_(1, at, q)
    q_bound = torch.zeros_like(p).scatter_add_(1, at, q * (grow + K * 2.0 ** -24))
    factor = c * t * grad_scale * weight.double()[:, None] * some[:, None]
    grad = factor * (p - scattered)
    p_bound = torch.where(p > 0, p * (err_sum + unit * torch.nan_to_num(zs, posinf=0.0)), 0.0)
    grad_bound = factor.abs() * (p_bound + q_bound + 4 * unit * (p + scattered) + 1e-37)
    loss = c * (weight.double() * row_loss).sum()
    loss_bound = c * (weight.double().abs() * (row_bound + (N / 32 + 40) * 2.0 ** -24 * row_loss.abs())).sum()
    return (row_loss, row_bound), (loss, loss_bound), (grad, grad_bound)


def close(name, got, want, bound):
    got = got.double()
    both = (got == want) | ((got - want).abs() <= bound)
    assert bool(both.all()), f"{name}: {got[~both][:4].tolist()} for {want[~both][:4].tolist()} +- {bound[~both][:4].tolist() if bound.dim() else bound}"


def inputs(rows, vocab, top, dtype, seed=0, index=torch.int64, values_dtype=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    teacher = torch.randn(rows, vocab, generator=gen, device="cuda") * 3
    values, indices = torch.topk(teacher, top, dim=1)
    student = (0.7 * teacher + torch.randn(rows, vocab, generator=gen, device="cuda")).to(dtype)
    weight = torch.rand(rows, generator=gen, device="cuda")
    return student, values.to(values_dtype or dtype), indices.to(index), weight


def run(student, values, indices, weight, temperature=1.0, grad=None, c=0.25, scale=None, op=None, health=None):
    N, V = student.shape
    grad = grad or student.dtype
    op = op or TopKDistillation(max(N, 1), V, values.shape[1])
    row_loss, loss = torch.full((N,), math.nan, device="cuda"), torch.full((1,), math.nan, device="cuda")
    ds = torch.full((N, V), math.nan, dtype=grad, device="cuda")
    factor = None if scale is None else torch.full((1,), scale, device="cuda")
    op.run(logits=student, teacher_values=values, teacher_indices=indices, temperature=temperature, row_weight=weight,
           loss_weight=c, row_loss=row_loss, loss_out=loss, dlogits=ds, grad_scale=factor, health=health)
    w = torch.ones(N, device="cuda") if weight is None else weight
    a, b, g = reference(student, values, indices, temperature, w, c, scale or 1.0)
    close("row_loss", row_loss, *a)
    close("loss", loss[0], *b)
    close("dlogits", ds, g[0], g[1] + U[grad] * g[0].abs() + ETA[grad])
    return row_loss, loss, ds


DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SIZES = [(1, 1, 1), (3, 2, 2), (7, 11, 3), (64, 101, 8), (33, 128, 128), (500, 257, 1), (20, 1024, 33), (9, 1025, 1000),
         (11, 2049, 64), (40, 5000, 1024), (5, 32768, 100), (300, 9001, 17), (3, 60001, 128), (2, 128257, 64), (1, 300000, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", SIZES)
def test_against_formulas(rows, vocab, top, dtype):
    run(*inputs(rows, vocab, top, dtype, seed=vocab), temperature=1.0 + (vocab % 3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grad", DTYPES)
@pytest.mark.parametrize("vocab", [100, 6003, 40002])
def test_types_of_the_gradient(dtype, grad, vocab):
    run(*inputs(13, vocab, 20, dtype, index=torch.int32, values_dtype=torch.float32), temperature=2.5, grad=grad, scale=64.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,top", [(297, 2049, 128), (310, 6144, 100), (300, 12301, 129), (301, 24001, 256), (299, 34990, 7),
                                            (300, 36000, 300), (1030, 3001, 12), (1100, 700, 20), (1201, 255, 40)])
def test_many_rows(rows, vocab, top, dtype):
    """Rows enough for every split of long rows over CTAs; absent and repeated entries, rows without weight, half of the
    tokens that are not the teacher's masked."""
    student, values, indices, weight = inputs(rows, vocab, top, dtype, seed=vocab)
    gen = torch.Generator(device="cuda").manual_seed(1)
    masked = torch.rand(rows, vocab, generator=gen, device="cuda") < 0.5
    masked.scatter_(1, indices, False)
    student = student.masked_fill(masked, -INF)
    indices = torch.where(torch.rand(rows, top, generator=gen, device="cuda") < 0.1, -1, indices)
    indices[:, top // 2] = indices[:, 0]
    weight = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.1, 0.0, weight)
    run(student, values, indices, weight, temperature=1.7, grad=torch.float32 if dtype == torch.bfloat16 else None)


@pytest.mark.parametrize("vocab", [60, 3000, 70000])
def test_absent_repeated_and_weightless(vocab):
    s, v, i, w = inputs(16, vocab, 12, torch.float32, seed=3)
    w[2], s[2, 5] = 0.0, math.nan  # a row of no weight is not read
    i[3] = -1                      # a row without a teacher
    i[4, 1:] = -1
    i[5, :6] = i[5, 0]             # a token repeated
    i[6, 3:9:2] = i[6, 4]
    v[7, 4:] = -INF
    v[8] = -INF
    v[9] = torch.finfo(torch.float32).min
    i[10], v[10] = vocab - 1, 1.0
    clean = s.clone()
    clean[2] = 0.0
    health = torch.zeros(1, dtype=torch.int32, device="cuda")
    row_loss, loss, ds = TopKDistillation(16, vocab, 12), None, None
    op = row_loss
    row_loss, loss = torch.empty(16, device="cuda"), torch.empty(1, device="cuda")
    ds = torch.full((16, vocab), math.nan, device="cuda")
    op.run(logits=s, teacher_values=v, teacher_indices=i, row_weight=w, row_loss=row_loss, loss_out=loss, dlogits=ds, health=health)
    a, b, g = reference(clean, v, i, 1.0, w, 1.0, 1.0)
    close("row_loss", row_loss, *a)
    close("loss", loss[0], *b)
    close("dlogits", ds, g[0], g[1] + U[torch.float32] * g[0].abs() + 1e-37)
    assert health.item() == 0
    for r in (2, 3, 8):
        assert row_loss[r] == 0 and not bool(ds[r].any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [70, 2500, 40000])
def test_masked_logits(vocab, dtype):
    s, v, i, w = inputs(8, vocab, 5, dtype, seed=4)
    low = torch.finfo(dtype).min
    keep = torch.zeros(8, vocab, dtype=torch.bool, device="cuda").scatter_(1, i, True)
    gone = ~keep & (torch.arange(vocab, device="cuda") % 2 == 0)
    s[:3] = torch.where(gone[:3], -INF, s[:3])
    s[3:5] = torch.where(gone[3:5], low, s[3:5])
    s[5] = -INF  # nothing left: no loss, no gradient
    s[6] = low
    row_loss, _, ds = run(s, v, i, w)
    assert row_loss[5] == 0 and not bool(ds[5].any())
    # a teacher's token that the student cannot choose: infinite loss, finite gradient
    s[7, i[7, 0]] = -INF
    op = TopKDistillation(8, vocab, 5)
    ds.zero_()
    op.run(logits=s, teacher_values=v, teacher_indices=i, row_loss=row_loss, dlogits=ds)
    assert row_loss[7] == INF and bool(torch.isfinite(ds).all())
    # NaN and +inf are not hidden, and stay in their rows
    s[0, 1], s[1, 2], v[2, 0] = math.nan, INF, math.nan
    op.run(logits=s, teacher_values=v, teacher_indices=i, row_loss=row_loss, dlogits=ds)
    assert bool(torch.isnan(row_loss[:3]).all()) and bool(torch.isnan(ds[:3]).any(1).all())
    assert bool(torch.isfinite(ds[3:]).all())


@pytest.mark.parametrize("vocab", [50, 4100, 33333])
def test_index_out_of_range_is_reported(vocab):
    s, v, i, w = inputs(6, vocab, 4, torch.float32)
    i[1, 2], i[4, 0] = vocab, 1 << 40
    health = torch.zeros(1, dtype=torch.int32, device="cuda")
    run(s, v, i, w, health=health)
    assert health.item() == 8


@pytest.mark.parametrize("vocab", [90, 3001, 50001])
def test_strides_and_alignments(vocab):
    s, v, i, w = inputs(7, vocab, 6, torch.bfloat16)
    want = run(s, v, i, w)
    wide_s = torch.full((7, vocab + 21), math.nan, dtype=torch.bfloat16, device="cuda")
    wide_g = torch.full((9, vocab + 10), 5.0, dtype=torch.bfloat16, device="cuda")
    wide_i = torch.full((7, 11), 1 << 50, device="cuda")
    for first in (0, 1, 5, 8):
        a, b = wide_s[:, first:first + vocab], wide_g[1:8, 3:3 + vocab]
        a.copy_(s)
        wide_i[:, 2:8] = i
        row_loss = torch.empty(7, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        TopKDistillation(7, vocab, 6).run(logits=a, teacher_values=v, teacher_indices=wide_i[:, 2:8], row_weight=w,
                                          loss_weight=0.25, row_loss=row_loss, dlogits=b, stream=side)
        side.synchronize()
        ref = reference(s, v, i, 1.0, w, 0.25, 1.0)
        close("row_loss", row_loss, *ref[0])
        close("dlogits", b, ref[2][0], ref[2][1] + U[torch.bfloat16] * ref[2][0].abs())
        assert bool((wide_g[0] == 5).all()) and bool((wide_g[8] == 5).all())
        assert bool((wide_g[:, :3] == 5).all()) and bool((wide_g[:, 3 + vocab:] == 5).all())
    assert bool(torch.isfinite(want[0]).all())


def test_loss_alone_repeats_and_graph():
    s, v, i, w = inputs(700, 3000, 10, torch.float32)
    op = TopKDistillation(1000, 3000, 10)
    first = run(s, v, i, w, op=op)
    again = run(s, v, i, w, op=op)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    loss = torch.zeros(1, device="cuda")
    op.run(logits=s, teacher_values=v, teacher_indices=i, row_weight=w, loss_weight=0.25, loss_out=loss)
    assert torch.equal(op.row_loss[:700], first[0]) and torch.equal(loss, first[1])
    graph = torch.cuda.CUDAGraph()
    loss.zero_()
    with torch.cuda.graph(graph):
        op.run(logits=s, teacher_values=v, teacher_indices=i, row_weight=w, loss_weight=0.25, loss_out=loss)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(loss, first[1])
    op.run(logits=s[:0], teacher_values=v[:0], teacher_indices=i[:0], loss_out=loss)
    assert loss.item() == 0


@pytest.mark.parametrize("vocab", [40, 3000])
def test_gradient_against_differences(vocab):
    """The gradient along a direction, against central differences of the loss in 64 bits."""
    s, v, i, w = inputs(4, vocab, 6, torch.float32, seed=8)
    _, _, ds = run(s, v, i, w, temperature=1.5)
    gen = torch.Generator(device="cuda").manual_seed(1)
    d = torch.randn(4, vocab, generator=gen, device="cuda", dtype=torch.float64)
    eps = 1e-4
    loss = lambda x: reference(x, v, i, 1.5, w, 0.25, 1.0)[1][0]  # noqa: E731
    slope = (loss(s.double() + eps * d) - loss(s.double() - eps * d)) / (2 * eps)
    bound = (reference(s, v, i, 1.5, w, 0.25, 1.0)[2][1] * d.abs()).sum() + 1e-6 * (1 + slope.abs())
    assert abs((ds.double() * d).sum() - slope) <= bound


def test_refusals():
    for args in ((0, 5, 1), (5, 0, 1), (5, 5, 0), (5, 5, 1025)):
        with pytest.raises(ValueError, match="must be positive"):
            TopKDistillation(*args)
    s, v, i, w = inputs(4, 50, 3, torch.float32)
    op = TopKDistillation(4, 50, 3)
    good = dict(logits=s, teacher_values=v, teacher_indices=i)

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            op.run(**{**good, **change})

    refused(ValueError, "logits must be", logits=s[:, :49])
    refused(ValueError, "logits must be", logits=s.double())
    refused(ValueError, "logits must be", logits=s.cpu())
    refused(ValueError, "contiguous rows", logits=torch.zeros(50, 4, device="cuda").t())
    refused(ValueError, "at most 4 rows", logits=torch.zeros(5, 50, device="cuda"))
    refused(ValueError, "teacher_values must be", teacher_values=v[:, :2])
    refused(ValueError, "teacher_indices must be", teacher_indices=i.to(torch.int16))
    refused(ValueError, "row_weight must be", row_weight=w[:3])
    refused(ValueError, "loss_out must be", loss_out=w)
    refused(ValueError, "dlogits must be", dlogits=s.double())
    refused(RuntimeError, "may not overwrite", dlogits=s)
    refused(RuntimeError, "temperature must be positive", temperature=0.0)
    refused(RuntimeError, "temperature must be positive", temperature=math.nan)
    refused(RuntimeError, "shorter than its row", logits=s[:1].expand(4, 50))
