"""Launches that begin while the stream's previous grid ends read what that grid wrote: chains of calls, each
reading the buffer that the call before has just written (and that held other values until then), give the
bits that the same calls give with a synchronisation between them."""

import pytest
import torch

from robolearn_b200.distillation import TopKDistillation
from robolearn_b200.gated import GatedMLP
from robolearn_b200.token_sampling import TokenSampler

pytestmark = pytest.mark.gpu


def _chain(calls, outputs, wait):
    kept = []
    for call, out in zip(calls, outputs):
        call()
        if wait:
            torch.cuda.synchronize()
        kept.append(out)
    copies = [k.clone() for k in kept]
    torch.cuda.synchronize()
    return copies


def _same(expected, got):
    assert len(expected) == len(got)
    for a, b in zip(expected, got):
        assert torch.isfinite(a).all() and a.abs().max() > 0
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_gated_blocks_read_what_the_call_before_wrote(rows):
    torch.manual_seed(0)
    width, depth = 256, 4
    block = GatedMLP(rows, width, width)
    weights = [(torch.randn(2, width, width, device="cuda") * 0.08).half() for _ in range(depth)]
    gradients = [(torch.empty_like(w[0]), torch.empty_like(w[1])) for w in weights]

    def run(wait):
        h = [torch.full((rows, width), float(i), device="cuda", dtype=torch.float16) for i in range(depth + 1)]
        d = [torch.full((rows, width), float(i), device="cuda", dtype=torch.float16) for i in range(depth + 1)]
        generator = torch.Generator("cuda").manual_seed(1)
        h[0].copy_(torch.randn(rows, width, device="cuda", generator=generator))
        d[depth].copy_(torch.randn(rows, width, device="cuda", generator=generator))
        torch.cuda.synchronize()
        calls = [lambda i=i: block.forward(x=h[i], gate_weight=weights[i][0], up_weight=weights[i][1], out=h[i + 1])
                 for i in range(depth)]
        calls += [lambda i=i: block.backward(x=h[i], gate_weight=weights[i][0], up_weight=weights[i][1], grad_out=d[i + 1],
                                             grad_x=d[i], grad_gate=gradients[i][0], grad_up=gradients[i][1])
                  for i in reversed(range(depth))]
        out = [h[i + 1] for i in range(depth)] + [d[i] for i in reversed(range(depth))]
        return _chain(calls, out, wait) + [g.clone() for pair in gradients for g in pair]

    _same(run(True), run(False))


@pytest.mark.parametrize("vocab", [101, 2000, 40000])
def test_sampling_and_distillation_read_what_the_call_before_wrote(vocab):
    torch.manual_seed(0)
    rows, top, steps = 64, 8, 12
    sampler, loss = TokenSampler(rows, vocab), TopKDistillation(rows, vocab, top)
    uniforms = torch.rand(rows, device="cuda")
    values = torch.randn(rows, top, device="cuda")
    indices = torch.randint(0, vocab, (rows, top), device="cuda", dtype=torch.int32)
    first = torch.randn(rows, vocab, device="cuda")

    def run(wait):
        # the gradient of one step is the logits of the next
        s = [first] + [torch.full((rows, vocab), float("nan"), device="cuda") for _ in range(steps)]
        tokens = [torch.zeros(rows, device="cuda", dtype=torch.int32) for _ in range(steps)]
        losses, row_loss = [torch.zeros(1, device="cuda") for _ in range(steps)], torch.empty(rows, device="cuda")
        torch.cuda.synchronize()
        calls, out = [], []
        for i in range(steps):
            calls.append(lambda i=i: loss.run(logits=s[i], teacher_values=values, teacher_indices=indices, row_loss=row_loss,
                                              dlogits=s[i + 1], loss_out=losses[i], loss_weight=100.0))
            calls.append(lambda i=i: sampler.run(logits=s[i + 1], uniforms=uniforms, tokens=tokens[i], top_k=50, top_p=0.9))
            out += [losses[i], tokens[i]]
        return _chain(calls, out, wait) + [x.clone() for x in s]

    _same(run(True), run(False))
