"""What is measured of the operators of a policy over discrete tokens: the gated feed-forward block of its
trunk (forward and backward), the distillation loss of its head from a teacher's top logits (with its
gradient), and drawing tokens from the head.

``run`` computes an operator in plain torch (32-bit arithmetic, rounded once at the end) where ``own`` is
false, and with this package's kernels where it is true."""

import math

import torch

own = False

ACTIVATIONS = ("silu", "gelu", "relu")
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
UNIT = float(2 ** 30)  # fixed-point unit of a token's weight


def listed():
    return [
        # acting: one environment's observation through the gated block of a 512-wide trunk
        dict(name="gated fwd one row", op="gated", backward=False, rows=1, features=512, hidden=2048, dtype="bf16", act="silu"),
        # acting: a few dozen environments, a wider trunk; the weights are most of what is read
        dict(name="gated fwd 48 rows", op="gated", backward=False, rows=48, features=2048, hidden=8192, dtype="fp16", act="gelu"),
        # a ragged minibatch of odd sizes (rows padded to 16 bytes, as operand planes are)
        dict(name="gated fwd ragged", op="gated", backward=False, rows=1777, features=523, hidden=1365, dtype="fp16", act="silu"),
        # the widest trunk of the repository (1024, times 4) over the rows of its largest batch (32768, both halves)
        dict(name="gated fwd 65536 rows", op="gated", backward=False, rows=65536, features=1024, hidden=4096, dtype="bf16", act="silu"),
        # training at the default batch (4096 transitions, both halves; 512-wide trunk, times 4)
        dict(name="gated bwd 8192 rows", op="gated", backward=True, rows=8192, features=512, hidden=2048, dtype="fp16", act="silu"),
        # training at the widest trunk and half of the largest batch's rows
        dict(name="gated bwd 32768 rows", op="gated", backward=True, rows=32768, features=1024, hidden=4096, dtype="bf16", act="gelu"),
        # a small head (the critic's 101 atoms) distilled from its teacher's eight best, fp32 as heads write it
        dict(name="distill 512 x 101", op="distill", rows=512, vocab=101, top=8, dtype="fp32", grad="fp32", temperature=1.0, masked=False),
        # a generic 32k vocabulary, fp32 logits, fp16 gradient for the next product, invalid tokens masked by -inf
        dict(name="distill 2048 x 32768", op="distill", rows=2048, vocab=32768, top=64, dtype="fp32", grad="fp16", temperature=2.0, masked=True),
        # a large vocabulary of odd size: rows start at any element
        dict(name="distill 2047 x 128257", op="distill", rows=2047, vocab=128257, top=128, dtype="bf16", grad="bf16", temperature=1.0, masked=False),
        # acting: 4096 environments, 256 action bins, nucleus only
        dict(name="sample 4096 x 256", op="sample", rows=4096, vocab=256, dtype="fp32", temperature=1.0, top_k=0, top_p=0.95, min_p=0.0, masked=True),
        # one request, large vocabulary: latency
        dict(name="sample 1 x 128257", op="sample", rows=1, vocab=128257, dtype="fp32", temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, masked=False),
        # a full batch of requests with every filter on
        dict(name="sample 256 x 131072", op="sample", rows=256, vocab=131072, dtype="bf16", temperature=0.9, top_k=2000, top_p=0.9, min_p=0.001, masked=False),
    ]


def draw(rng):
    def spread(low, high):
        n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
        return n + 1 if n == 3072 else n

    op = rng.choice(("gated", "gated", "distill", "sample"))
    if op == "gated":
        backward = rng.random() < 0.5
        features, hidden = spread(64, 2048), spread(64, 8192)
        most = (32768 if backward else 65536) * 1024 * 4096
        return dict(op="gated", backward=backward, rows=spread(1, max(1, min(65536, most // (features * hidden)))),
                    features=features, hidden=hidden, dtype=rng.choice(("fp16", "bf16")), act=rng.choice(ACTIVATIONS))
    if op == "distill":
        vocab = spread(11, 160000)
        dtype = rng.choice(("fp32", "fp16", "bf16"))
        return dict(op="distill", rows=spread(1, min(16384, 250_000_000 // (vocab * SIZE[dtype] // 2))), vocab=vocab,
                    top=spread(1, min(vocab, 256)), dtype=dtype, grad=rng.choice((dtype, "fp16")),
                    temperature=round(rng.uniform(0.5, 4.0), 3), masked=vocab > 64 and rng.random() < 0.5)
    vocab = spread(2, 200000)
    return dict(op="sample", rows=spread(1, min(8192, 33_000_000 // vocab)), vocab=vocab,
                dtype=rng.choice(("fp32", "fp16", "bf16")), temperature=round(rng.uniform(0.3, 2.0), 3),
                top_k=rng.choice((0, spread(1, vocab))), top_p=rng.choice((1.0, round(rng.uniform(0.1, 0.99), 3))),
                min_p=rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.3), 4))), masked=vocab > 64 and rng.random() < 0.5)


def padded(shape, dtype, values=None):
    """A matrix whose rows start on 16-byte boundaries (a view of a wider one, as the operand planes are)."""
    rows, cols = shape
    full = torch.zeros(rows, (cols + 7) // 8 * 8, dtype=dtype, device="cuda")
    view = full[:, :cols]
    if values is not None:
        view.copy_(values)
    return view


def prepare(case, seed):
    """The inputs, from the seed alone; the output buffers; and the operator's handle where the package has one."""
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] == "gated":
        m, k, f, dt = case["rows"], case["features"], case["hidden"], DTYPES[case["dtype"]]
        s["x"] = padded((m, k), dt, normal(m, k))
        # rows of unit length, as the trunk's projected weights are, times sqrt(2) for the activations' size
        s["wg"] = padded((f, k), dt, normal(f, k) * math.sqrt(2.0 / k))
        s["wu"] = padded((f, k), dt, normal(f, k) * math.sqrt(2.0 / k))
        if case["backward"]:
            s["dh"] = padded((m, f), dt, normal(m, f))
            s["dx"], s["dwg"], s["dwu"] = padded((m, k), dt), padded((f, k), dt), padded((f, k), dt)
        else:
            s["h"] = padded((m, f), dt)
        if own:
            from robolearn_b200.gated import GatedMLP

            s["op"] = GatedMLP(m, k, f, dtype=dt, activation=case["act"])
    elif case["op"] == "distill":
        n, v, top, dt = case["rows"], case["vocab"], case["top"], DTYPES[case["dtype"]]
        teacher = normal(n, v) * 3.0
        if case["masked"]:
            gone = torch.rand(v, generator=gen, device="cuda") < 0.1
            gone[0] = False
            teacher.masked_fill_(gone, -math.inf)
        values, s["indices"] = torch.topk(teacher, top, dim=1)
        s["values"] = values.to(dt)
        s["logits"] = teacher.mul_(0.8).add_(normal(n, v)).to(dt)
        del teacher, values
        # a teacher that answered with fewer entries, and rows of padding
        s["indices"].masked_fill_(torch.rand(n, top, generator=gen, device="cuda") < 0.02, -1)
        s["weight"] = (torch.rand(n, generator=gen, device="cuda") < 0.95).float()
        s["row_loss"], s["loss"] = torch.empty(n, device="cuda"), torch.empty(1, device="cuda")
        s["dlogits"] = torch.empty(n, v, dtype=DTYPES[case["grad"]], device="cuda")
        # the loss scale that fp16 gradients are kept at
        s["scale"] = torch.full((1,), 32.0 * n, device="cuda") if case["grad"] == "fp16" else None
        if own:
            from robolearn_b200.distillation import TopKDistillation

            s["op"] = TopKDistillation(n, v, top)
    else:
        r, v, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
        logits = normal(r, v) * 3.0
        if case["masked"]:
            logits.masked_fill_(torch.rand(r, v, generator=gen, device="cuda") < 0.1, -math.inf)
            logits[r // 2] = -math.inf  # a row that its mask leaves empty
        s["logits"] = logits.to(dt)
        s["uniforms"] = torch.rand(r, generator=gen, device="cuda")
        s["tokens"] = torch.empty(r, dtype=torch.int32, device="cuda")
        s["log_probs"] = torch.empty(r, device="cuda")
        if own:
            from robolearn_b200.token_sampling import TokenSampler

            s["op"] = TokenSampler(r, v)
    return s


def act_and_slope(name, g):
    """The activation and its derivative."""
    if name == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    if name == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    return g.clamp(min=0.0), (g > 0).to(g.dtype)


def gated_plain(s):
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a, slope = act_and_slope(s["case"]["act"], g)
    if not s["case"]["backward"]:
        return {"h": a * u}
    dh = s["dh"].float()
    dg, du = dh * u * slope, dh * a
    return {"dx": dg @ wg + du @ wu, "dwg": dg.t() @ x, "dwu": du.t() @ x}


def distill_plain(s):
    c = s["case"]
    t = c["temperature"]
    n = c["rows"]
    here = s["indices"] >= 0
    at = s["indices"].clamp(min=0)
    tz = torch.where(here, s["values"].float() / t, -math.inf)
    top = tz.amax(1, keepdim=True)
    e = torch.where(top > -math.inf, torch.exp(tz - top), 0.0)
    total = e.sum(1, keepdim=True)
    q = torch.where(total > 0, e / total, 0.0)
    z = s["logits"].float() / t
    z = z - z.amax(1, keepdim=True)
    p = torch.exp(z)
    total_p = p.sum(1, keepdim=True)
    log_q = torch.log(torch.where(q > 0, q, 1.0))
    log_p = z.gather(1, at) - torch.log(total_p)
    row_loss = (t * t) * torch.where(q > 0, q * (log_q - log_p), 0.0).sum(1)
    weight = s["weight"]
    row_loss = torch.where(weight != 0, row_loss, 0.0)
    p = p / total_p
    p.scatter_add_(1, at, -q)
    # a row with no teacher entry, or of no weight, has no gradient
    factor = torch.where(total[:, 0] > 0, weight * (t / n), 0.0)[:, None]
    if s["scale"] is not None:
        factor = factor * s["scale"]
    return {"row_loss": row_loss, "loss": (weight * row_loss).sum().reshape(1) / n, "dlogits": (factor * p).to(DTYPES[c["grad"]])}


def sample_plain(s):
    c = s["case"]
    v = c["vocab"]
    x = s["logits"].float()
    best = x.amax(1, keepdim=True)
    empty = best == -math.inf
    inverse = torch.ones((), device="cuda") / torch.tensor(c["temperature"], device="cuda")
    e = torch.exp(torch.where(empty, -math.inf, (x - best) * inverse))
    weight = torch.round(e * UNIT).to(torch.int64)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ranked = weight.gather(1, order)
    if 0 < c["top_k"] < v:
        ranked[:, c["top_k"]:] = 0
    before = ranked.cumsum(1) - ranked
    keep = before.double() < torch.tensor(c["top_p"], device="cuda").double() * ranked.sum(1, keepdim=True).double()
    if c["top_p"] >= 1.0:
        keep = torch.ones_like(keep)
    keep[:, 0] = True
    kept = torch.zeros_like(weight).scatter_(1, order, torch.where(keep, ranked, 0))
    kept = torch.where(e >= torch.tensor(c["min_p"], device="cuda"), kept, 0)
    total = kept.sum(1, keepdim=True)
    target = torch.minimum((s["uniforms"].double()[:, None] * total.double()).to(torch.int64), total - 1)
    token = (kept.cumsum(1) > target).to(torch.int32).argmax(1, keepdim=True)
    mine = kept.gather(1, token)
    share = mine.to(e.dtype) / total.to(e.dtype)
    log_prob = torch.where(share > 0.5, torch.log1p(-(total - mine).to(e.dtype) / total.to(e.dtype)), torch.log(share))
    return {"tokens": torch.where(empty, -1, token)[:, 0].to(torch.int32),
            "log_probs": torch.where(empty, -math.inf, log_prob)[:, 0]}


def run(s):
    c = s["case"]
    if c["op"] == "gated":
        if own:
            if c["backward"]:
                s["op"].backward(x=s["x"], gate_weight=s["wg"], up_weight=s["wu"], grad_out=s["dh"],
                                 grad_x=s["dx"], grad_gate=s["dwg"], grad_up=s["dwu"])
                return {"dx": s["dx"], "dwg": s["dwg"], "dwu": s["dwu"]}
            s["op"].forward(x=s["x"], gate_weight=s["wg"], up_weight=s["wu"], out=s["h"])
            return {"h": s["h"]}
        return {k: v.to(s["x"].dtype) for k, v in gated_plain(s).items()}
    if c["op"] == "distill":
        if own:
            s["op"].run(logits=s["logits"], teacher_values=s["values"], teacher_indices=s["indices"],
                        temperature=c["temperature"], row_weight=s["weight"], loss_weight=1.0 / c["rows"],
                        row_loss=s["row_loss"], loss_out=s["loss"], dlogits=s["dlogits"], grad_scale=s["scale"])
            return {"row_loss": s["row_loss"], "loss": s["loss"], "dlogits": s["dlogits"]}
        return distill_plain(s)
    if own:
        s["op"].run(logits=s["logits"], uniforms=s["uniforms"], tokens=s["tokens"], log_probs=s["log_probs"],
                    temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])
        return {"tokens": s["tokens"], "log_probs": s["log_probs"]}
    return sample_plain(s)


def exact(case, seed):
    """The same outputs from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "gated":
        x, wg, wu = s["x"].double(), s["wg"].double(), s["wu"].double()
        g = torch.einsum("mk,fk->mf", x, wg)
        if case["act"] == "silu":
            a, slope = g * torch.sigmoid(g), torch.sigmoid(g) + g * torch.sigmoid(g) * torch.sigmoid(-g)
        elif case["act"] == "gelu":
            cdf = torch.special.ndtr(g)
            a, slope = g * cdf, cdf + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
        else:
            a, slope = torch.relu(g), torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))
        u = torch.einsum("mk,fk->mf", x, wu)
        if not case["backward"]:
            return {"h": a * u}
        dh = s["dh"].double()
        dg = dh * u * slope
        du = dh * a
        return {"dx": torch.einsum("mf,fk->mk", dg, wg) + torch.einsum("mf,fk->mk", du, wu),
                "dwg": torch.einsum("mf,mk->fk", dg, x), "dwu": torch.einsum("mf,mk->fk", du, x)}
    if case["op"] == "distill":
        t, n = case["temperature"], case["rows"]
        row_loss = torch.zeros(n, dtype=torch.float64, device="cuda")
        grad = torch.zeros(n, case["vocab"], dtype=torch.float64, device="cuda")
        scale = 1.0 if s["scale"] is None else float(s["scale"])
        for r in range(0, n, 512):
            rows = slice(r, r + 512)
            index, weight = s["indices"][rows], s["weight"][rows].double()
            student = torch.log_softmax(s["logits"][rows].double() / t, 1)
            teacher = torch.log_softmax((s["values"][rows].double() / t).masked_fill(index < 0, -math.inf), 1)
            q = torch.nan_to_num(teacher.exp(), nan=0.0)
            index = index.clamp(min=0)
            cross = q * (torch.nan_to_num(teacher, nan=0.0, neginf=0.0) - student.gather(1, index))
            row_loss[rows] = t * t * torch.where((q > 0) & (weight != 0)[:, None], cross, 0.0).sum(1)
            some = (q.sum(1) > 0) * weight * t * scale / n
            grad[rows] = some[:, None] * (student.exp() - torch.zeros_like(student).scatter_add_(1, index, q))
        return {"row_loss": row_loss, "loss": (row_loss * s["weight"].double()).sum().reshape(1) / n, "dlogits": grad}
    tokens, log_probs = [], []
    k, v = case["top_k"], case["vocab"]
    t, top_p, min_p = (float(torch.tensor(case[name])) for name in ("temperature", "top_p", "min_p"))  # as 32 bits hold them
    for r in range(0, case["rows"], 64):
        x = s["logits"][r:r + 64].double()
        best = x.amax(1, keepdim=True)
        empty = (best == -math.inf)[:, 0]
        e = torch.exp((x - best.clamp(min=-1e300)) / t)
        order = torch.argsort(x, dim=1, descending=True, stable=True)
        rank = torch.empty_like(order).scatter_(1, order, torch.arange(v, device="cuda").expand_as(order))
        held = torch.where(rank < k, e, 0.0) if 0 < k < v else e
        ahead = held.gather(1, order).cumsum(1).gather(1, rank) - held  # mass of the tokens before each one
        if top_p < 1.0:
            held = torch.where((ahead < top_p * held.sum(1, keepdim=True)) | (rank == 0), held, 0.0)
        held = torch.where(e >= min_p, held, 0.0)
        sums = held.cumsum(1)
        drawn = torch.searchsorted(sums, s["uniforms"][r:r + 64].double()[:, None] * sums[:, -1:], right=True).clamp(max=v - 1)
        share = held.gather(1, drawn) / sums[:, -1:]
        tokens.append(torch.where(empty, -1, drawn[:, 0]))
        log_probs.append(torch.where(empty, -math.inf, share[:, 0].log()))
    return {"tokens": torch.cat(tokens).to(torch.int32), "log_probs": torch.cat(log_probs)}


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once."""
    if case["op"] == "gated":
        m, k, f = case["rows"], case["features"], case["hidden"]
        moved = 2 * (m * k + 2 * f * k + m * f)
        if case["backward"]:  # the two projections again, two products for dx, two for the weights
            return {"bytes": moved + 2 * (m * k + 2 * f * k), "flops": 12 * m * k * f}
        return {"bytes": moved, "flops": 4 * m * k * f}
    if case["op"] == "distill":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * (v * (SIZE[case["dtype"]] + SIZE[case["grad"]]) + case["top"] * (SIZE[case["dtype"]] + 8) + 8),
                "flops": 6 * n * v}
    return {"bytes": case["rows"] * (case["vocab"] * SIZE[case["dtype"]] + 12), "flops": 4 * case["rows"] * case["vocab"]}
