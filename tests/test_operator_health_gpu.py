"""The operators refuse a health word that the device cannot write: one in host memory, one of another type. Nothing is
launched."""

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.distillation import TopKDistillation  # noqa: E402
from robolearn_b200.gated import GatedMLP  # noqa: E402
from robolearn_b200.token_sampling import TokenSampler  # noqa: E402


def _calls():
    x, w = torch.randn(4, 16, device="cuda").half(), torch.randn(16, 16, device="cuda").half()
    h, dx = torch.full_like(x, 7.0), torch.full_like(x, 7.0)
    block = GatedMLP(4, 16, 16)
    logits, tokens = torch.randn(4, 50, device="cuda"), torch.full((4,), 7, dtype=torch.int32, device="cuda")
    values, indices, ds = torch.zeros(4, 2, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"), torch.full((4, 50), 7.0, device="cuda")
    yield h, lambda health: block.forward(x=x, gate_weight=w, up_weight=w, out=h, health=health)
    yield dx, lambda health: block.backward(x=x, gate_weight=w, up_weight=w, grad_out=h, grad_x=dx, health=health)
    yield tokens, lambda health: TokenSampler(4, 50).run(logits=logits, uniforms=torch.zeros(4, device="cuda"), tokens=tokens, health=health)
    yield ds, lambda health: TopKDistillation(4, 50, 2).run(logits=logits, teacher_values=values, teacher_indices=indices, dlogits=ds, health=health)


def test_health_word():
    for out, call in _calls():
        before = out.clone()
        for bad in (torch.zeros(1, dtype=torch.int32), torch.zeros(1, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda"),
                    torch.zeros(0, dtype=torch.int32, device="cuda")):
            with pytest.raises(ValueError, match="health must be"):
                call(bad)
        torch.cuda.synchronize()
        assert torch.equal(out, before)
        for good in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros((), dtype=torch.int32, device="cuda"),
                     torch.zeros(4, dtype=torch.int32, device="cuda")):
            call(good)
            assert not bool(good.any())
        assert not torch.equal(out, before)
