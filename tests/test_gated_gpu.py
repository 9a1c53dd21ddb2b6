"""Gated feed-forward block (``rl2_gated_*``) against the formulas in 64 bits.

Bounds, per element, with u the unit roundoff of the 16-bit type (2^-11 fp16, 2^-8 bf16), eta its
smallest subnormal's half and a the relative size of a product sum's accumulation error (1e-8 per
term: the tensor cores' fp32 accumulation, measured at 7e-9, plus the rest of the fp32 arithmetic):
  g, u_        a_K S      with S the sum of |products|
  h            u |h| + eta + the errors of g and u_ through the formula
  dg, du       one rounding (u, eta) before the last products, so those carry
               u (|dg| |Wg| + |du| |Wu|) and their own accumulation error."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.dense import operand_ld  # noqa: E402
from robolearn_b200.gated import ACTIVATIONS, GatedMLP  # noqa: E402

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ETA = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
PER_TERM = 1e-8


def act64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2.0)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    return g.clamp(min=0), (g > 0).to(g.dtype)


def matrix(rows, cols, dtype, gen=None, scale=1.0, extra=0, fill=float("nan")):
    """[rows, cols] view of rows padded to 16 bytes (plus ``extra`` elements); the padding holds NaN."""
    full = torch.full((max(rows, 1), operand_ld(cols, 0) + extra), fill, dtype=dtype, device="cuda")
    view = full[:rows, :cols]
    if gen is not None:
        view.copy_(torch.randn(rows, cols, generator=gen, device="cuda") * scale)
    return view


def inputs(rows, features, hidden, dtype, extra=0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = matrix(rows, features, dtype, gen, 1.0, extra)
    wg = matrix(hidden, features, dtype, gen, 1 / math.sqrt(features), extra)
    wu = matrix(hidden, features, dtype, gen, 1 / math.sqrt(features))
    dh = matrix(rows, hidden, dtype, gen, 1.0, extra)
    return x, wg, wu, dh


def reference(x, wg, wu, dh, act):
    """Outputs and their bounds' parts, in 64 bits."""
    dt = x.dtype
    u, eta, K = U[dt], ETA[dt], x.shape[1]
    x, wg, wu, dh = x.double(), wg.double(), wu.double(), dh.double()
    g, up = x @ wg.t(), x @ wu.t()
    eg = (PER_TERM * K + 1e-6) * (x.abs() @ wg.abs().t())
    eu = (PER_TERM * K + 1e-6) * (x.abs() @ wu.abs().t())
    a, slope = act64(act, g)
    lip = 1.13  # max |act'| of the three activations
    bend = 0.8 if act != "relu" else 0.0  # max |act''| (ReLU: no kink is crossed away from g = 0, see the caller)
    out = {"h": (a * up, u * (a * up).abs() + eta + 1.01 * (lip * eg * (up.abs() + eu) + a.abs() * eu + 1e-6 * (a * up).abs()))}
    dg, du = dh * up * slope, dh * a
    edg = u * dg.abs() + eta + 1.01 * dh.abs() * (eu * lip + (up.abs() + eu) * (bend * eg + 1e-6))
    if act == "relu":  # a gate within its error of the kink may fall on either side
        edg = edg + torch.where(g.abs() <= eg, (dh * up).abs(), 0.0)
    edu = u * du.abs() + eta + 1.01 * dh.abs() * (lip * eg + 1e-6 * a.abs())
    both = lambda p, q, r, s: p @ r + q @ s  # noqa: E731
    F, M = wg.shape[0], x.shape[0]
    size = both(dg.abs(), du.abs(), wg.abs(), wu.abs())
    dx = dg @ wg + du @ wu
    out["dx"] = (dx, 1.01 * (both(edg, edu, wg.abs(), wu.abs()) + (PER_TERM * 2 * F + 1e-6) * size) + u * dx.abs() + eta)
    for name, d, e in (("dwg", dg, edg), ("dwu", du, edu)):
        w = d.t() @ x
        out[name] = (w, 1.01 * (e.t() @ x.abs() + (PER_TERM * M + 1e-6) * (d.abs().t() @ x.abs())))
    return out


def check(name, got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{name}: off by up to {(off / bound).max().item():.2f} of the bound"


def run(rows, features, hidden, dtype, act, extra=0, weight_dtype=None, plan_rows=None):
    x, wg, wu, dh = inputs(rows, features, hidden, dtype, extra)
    op = GatedMLP(plan_rows or max(rows, 1), features, hidden, dtype=dtype, activation=act)
    h, dx = matrix(rows, hidden, dtype, extra=extra), matrix(rows, features, dtype)
    wt = weight_dtype or dtype
    dwg, dwu = matrix(hidden, features, wt), matrix(hidden, features, wt, extra=extra)
    health = torch.zeros(1, dtype=torch.int32, device="cuda")
    op.forward(x=x, gate_weight=wg, up_weight=wu, out=h, health=health)
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx, grad_gate=dwg, grad_up=dwu, health=health)
    assert health.item() == 0
    ref = reference(x, wg, wu, dh, act)
    check("h", h, *ref["h"])
    check("dx", dx, *ref["dx"])
    for name, t in (("dwg", dwg), ("dwu", dwu)):
        want, bound = ref[name]
        if wt == dtype:
            bound = bound + U[dtype] * want.abs() + ETA[dtype]
        check(name, t, want, bound)
    return h, dx, dwg, dwu


SIZES = [(1, 1, 1), (1, 64, 128), (2, 8, 3), (5, 512, 96), (7, 100, 1000), (8, 16, 17), (9, 2048, 640), (16, 500, 257), (17, 136, 72), (33, 1000, 40),
         (64, 64, 64), (65, 520, 260), (100, 31, 333), (128, 256, 128), (129, 72, 200), (200, 1024, 1024), (257, 523, 1365),
         (777, 65, 63), (1500, 256, 512), (4097, 129, 130)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,features,hidden", SIZES)
def test_against_formulas(rows, features, hidden, dtype):
    acts = sorted(ACTIVATIONS)
    run(rows, features, hidden, dtype, acts[(rows + hidden) % 3])


@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
@pytest.mark.parametrize("rows", [3, 300])
def test_every_activation(act, rows):
    run(rows, 256, 384, torch.bfloat16, act)
    run(rows, 256, 384, torch.float16, act, extra=24, plan_rows=400)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,features,hidden", [(1, 40, 24), (130, 257, 300), (9000, 64, 256)])
def test_fp32_weight_gradients(rows, features, hidden, dtype):
    """Including contractions long enough to be split over the rows."""
    run(rows, features, hidden, dtype, "silu", weight_dtype=torch.float32)


@pytest.mark.parametrize("rows,features,hidden,dtype", [(40, 64, 96, torch.float16), (17000, 64, 128, torch.float16)])
def test_scaled_weight_gradients(rows, features, hidden, dtype):
    """A power of two before the rounding: the same bits, scaled (also where the rows are split)."""
    x, wg, wu, dh = inputs(rows, features, hidden, dtype)
    op = GatedMLP(rows, features, hidden, dtype=dtype)
    make = lambda: (matrix(hidden, features, torch.float32), matrix(hidden, features, torch.float32))  # noqa: E731
    a, b = make()
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_gate=a, grad_up=b)
    c, d = make()
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_gate=c, grad_up=d,
                grad_weight_scale=torch.full((1,), 2.0 ** -10, device="cuda"))
    assert torch.equal(c * 1024, a) and torch.equal(d * 1024, b)


def test_outputs_stay_inside():
    """The padding between rows (poisoned with NaN on input) is neither read nor written."""
    x, wg, wu, _ = inputs(70, 77, 83, torch.float16, extra=16)
    op = GatedMLP(70, 77, 83)
    full = torch.full((72, 104), 5.0, dtype=torch.float16, device="cuda")
    op.forward(x=x, gate_weight=wg, up_weight=wu, out=full[1:71, :83])
    assert bool((full[0] == 5).all()) and bool((full[71] == 5).all()) and bool((full[:, 83:] == 5).all())
    assert bool(torch.isfinite(full).all())


def test_not_finite_values_stay_in_their_rows():
    x, wg, wu, dh = inputs(40, 64, 96, torch.bfloat16)
    op = GatedMLP(40, 64, 96, dtype=torch.bfloat16)
    clean, h = matrix(40, 96, torch.bfloat16), matrix(40, 96, torch.bfloat16)
    op.forward(x=x, gate_weight=wg, up_weight=wu, out=clean)
    x[7, 3], x[21, 0] = float("nan"), float("inf")
    op.forward(x=x, gate_weight=wg, up_weight=wu, out=h)
    keep = torch.ones(40, dtype=torch.bool, device="cuda")
    keep[[7, 21]] = False
    assert torch.equal(h[keep], clean[keep])
    assert bool(torch.isnan(h[7]).all()) and not bool(torch.isfinite(h[21]).all())


def test_no_rows():
    wg, wu = matrix(24, 16, torch.float16, fill=1.0), matrix(24, 16, torch.float16, fill=1.0)
    op = GatedMLP(4, 16, 24)
    x, h = matrix(0, 16, torch.float16), matrix(0, 24, torch.float16)
    dwg, dwu = matrix(24, 16, torch.float32), matrix(24, 16, torch.float32)
    op.forward(x=x, gate_weight=wg, up_weight=wu, out=h)
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=h, grad_x=x, grad_gate=dwg, grad_up=dwu)
    assert not bool(dwg.any()) and not bool(dwu.any())


def test_parts_of_the_backward_and_repeatability():
    """grad_x alone, the weight gradients alone and all together agree bit for bit, and so do repeats."""
    x, wg, wu, dh = inputs(2100, 200, 328, torch.bfloat16)
    op = GatedMLP(4096, 200, 328, dtype=torch.bfloat16)
    make = lambda: (matrix(2100, 200, torch.bfloat16), matrix(328, 200, torch.float32), matrix(328, 200, torch.float32))  # noqa: E731
    dx, dwg, dwu = make()
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx, grad_gate=dwg, grad_up=dwu)
    dx2, dwg2, dwu2 = make()
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx2)
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_gate=dwg2, grad_up=dwu2)
    assert torch.equal(dx, dx2) and torch.equal(dwg, dwg2) and torch.equal(dwu, dwu2)


def test_other_stream_and_graph():
    x, wg, wu, dh = inputs(300, 128, 256, torch.float16)
    op = GatedMLP(300, 128, 256)
    op.workspace()
    h, dx = matrix(300, 256, torch.float16), matrix(300, 128, torch.float16)
    dwg, dwu = matrix(256, 128, torch.float16), matrix(256, 128, torch.float16)

    def both(stream=None):
        op.forward(x=x, gate_weight=wg, up_weight=wu, out=h, stream=stream)
        op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx, grad_gate=dwg, grad_up=dwu, stream=stream)

    both()
    want = [t.clone() for t in (h, dx, dwg, dwu)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for t in (h, dx, dwg, dwu):
        t.zero_()
    side.wait_stream(torch.cuda.current_stream())
    both(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((h, dx, dwg, dwu), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for t in (h, dx, dwg, dwu):
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((h, dx, dwg, dwu), want))


@pytest.mark.parametrize("act", sorted(ACTIVATIONS))
def test_gradients_against_differences(act):
    """d sum(h dh) along a direction from the backward, against central differences of the formula in
    64 bits: the differences' own error is O(eps^2) = 1e-10, the gradients' is their bound."""
    x, wg, wu, dh = inputs(3, 24, 40, torch.float16, seed=3)
    op = GatedMLP(3, 24, 40, activation=act)
    dx, dwg, dwu = matrix(3, 24, torch.float16), matrix(40, 24, torch.float32), matrix(40, 24, torch.float32)
    op.backward(x=x, gate_weight=wg, up_weight=wu, grad_out=dh, grad_x=dx, grad_gate=dwg, grad_up=dwu)
    ref = reference(x, wg, wu, dh, act)
    p = [t.double() for t in (x, wg, wu)]
    gen = torch.Generator(device="cuda").manual_seed(9)

    def loss(q):
        return (act64(act, q[0] @ q[1].t())[0] * (q[0] @ q[2].t()) * dh.double()).sum()

    for i, (name, grad) in enumerate((("dx", dx), ("dwg", dwg), ("dwu", dwu))):
        v = torch.randn(p[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        eps = 1e-5
        plus, minus = list(p), list(p)
        plus[i], minus[i] = p[i] + eps * v, p[i] - eps * v
        slope = (loss(plus) - loss(minus)) / (2 * eps)
        bound = (ref[name][1] * v.abs()).sum() + 1e-6 * (1 + slope.abs())
        assert abs((grad.double() * v).sum() - slope) <= bound, name


def test_refusals():
    with pytest.raises(ValueError, match="fp16 or bf16"):
        GatedMLP(4, 16, 16, dtype=torch.float32)
    with pytest.raises(ValueError, match="activation"):
        GatedMLP(4, 16, 16, activation="tanh")
    with pytest.raises(RuntimeError, match="positive"):
        GatedMLP(0, 16, 16)
    op = GatedMLP(4, 16, 24)
    x, wg, wu, dh = inputs(4, 16, 24, torch.float16)
    h = matrix(4, 24, torch.float16)
    good = dict(x=x, gate_weight=wg, up_weight=wu, out=h)

    def refused(error, match, **change):
        with pytest.raises(error, match=match):
            op.forward(**{**good, **change})

    refused(ValueError, "shape", x=x[:, :15])
    refused(ValueError, "must be torch.float16", x=x.bfloat16())
    refused(ValueError, "must be on", gate_weight=wg.cpu())
    refused(ValueError, "contiguous rows", up_weight=torch.zeros(16, 24, dtype=torch.float16, device="cuda").t())
    refused(RuntimeError, "multiple of 16 bytes", x=torch.zeros(4, 17, dtype=torch.float16, device="cuda")[:, :16])
    refused(RuntimeError, "16-byte aligned", x=torch.zeros(4, 24, dtype=torch.float16, device="cuda")[:, 1:17])
    refused(RuntimeError, "rows must be", x=torch.zeros(5, 16, dtype=torch.float16, device="cuda"),
            out=torch.zeros(5, 24, dtype=torch.float16, device="cuda"))
    back = dict(x=x, gate_weight=wg, up_weight=wu, grad_out=dh)
    with pytest.raises(RuntimeError, match="no gradient"):
        op.backward(**back)
    with pytest.raises(ValueError, match="come together"):
        op.backward(**back, grad_gate=matrix(24, 16, torch.float16))
    with pytest.raises(ValueError, match="grad_weight_scale must be"):
        op.backward(**back, grad_gate=matrix(24, 16, torch.float16), grad_up=matrix(24, 16, torch.float16), grad_weight_scale=dh)
    with pytest.raises(RuntimeError, match="may not be x"):
        op.backward(**back, grad_x=x)
