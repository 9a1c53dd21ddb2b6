"""Buffers that the operators keep (the distillation's counter and row losses, the gated block's workspace), on streams
other than the one that made them."""

import gc

import pytest
import torch

pytestmark = pytest.mark.gpu

from robolearn_b200.distillation import TopKDistillation  # noqa: E402
from robolearn_b200.gated import GatedMLP  # noqa: E402

CYCLES = 200_000_000  # about a tenth of a second


def _distillation_inputs(rows, vocab):
    gen = torch.Generator(device="cuda").manual_seed(0)
    logits = torch.randn(rows, vocab, generator=gen, device="cuda")
    values, indices = torch.topk(logits + torch.randn(rows, vocab, generator=gen, device="cuda"), 4, dim=1)
    return dict(logits=logits, teacher_values=values, teacher_indices=indices)


def _block(rows=300, width=512):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, wg, wu, dh = (torch.randn(n, width, generator=gen, device="cuda").half() * 0.1 for n in (rows, width, width, rows))
    return dict(x=x, gate_weight=wg, up_weight=wu, grad_out=dh), GatedMLP(rows, width, width)


@pytest.mark.parametrize("given", [True, False])
def test_counter_is_clear_before_a_call_on_another_stream(given):
    """The object is made while its stream is busy, and called at once on another: the total is written."""
    inputs = _distillation_inputs(64, 90)
    want, got = torch.zeros(1, device="cuda"), torch.full((1,), float("nan"), device="cuda")
    TopKDistillation(64, 90, 4).run(**inputs, loss_out=want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    poisoned = [torch.full((1,), 12345, dtype=torch.int32, device="cuda") for _ in range(256)]  # what the counter's memory may hold
    torch.cuda.synchronize()
    del poisoned
    torch.cuda._sleep(CYCLES)
    op = TopKDistillation(64, 90, 4)
    if given:
        op.run(**inputs, loss_out=got, stream=side)
    else:
        with torch.cuda.stream(side):
            op.run(**inputs, loss_out=got)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and op.counter.item() == 0


@pytest.mark.parametrize("given", [True, False])
def test_buffers_are_not_reused_under_another_stream(given):
    """An operator that is dropped while a side stream still works: its memory goes to nobody else until that is done."""
    side = torch.cuda.Stream()

    def on_side(call):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(CYCLES)
            if not given:
                call()
        if given:
            call(stream=side)

    def reused(size, address):
        gc.collect()
        assert not side.query()
        fresh = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(4)]
        assert not side.query()
        return any(t.data_ptr() == address for t in fresh)

    rows = 5_000_000  # row losses of 20 MB: a block of their own
    inputs = _distillation_inputs(8, 90)
    op = TopKDistillation(rows, 90, 4)
    on_side(lambda **k: op.run(**inputs, **k))
    address, size = op.row_loss.data_ptr(), rows * 4
    del op
    assert not reused(size, address)
    torch.cuda.synchronize()

    inputs, op = _block()
    dx = torch.empty_like(inputs["x"])
    address, size = op.workspace().data_ptr(), op.workspace_bytes()
    on_side(lambda **k: op.backward(**inputs, grad_x=dx, **k))
    del op
    assert not reused(size, address)
    torch.cuda.synchronize()


def test_workspace_memory_is_free_when_it_is_taken():
    """The workspace's memory may come from a tensor that its stream is not done with: by the time it is handed out,
    that stream is."""
    inputs, op = _block()
    want, got = torch.empty_like(inputs["x"]), torch.empty_like(inputs["x"])
    GatedMLP(300, 512, 512).backward(**inputs, grad_x=want)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    earlier = torch.empty(op.workspace_bytes(), dtype=torch.uint8, device="cuda")
    torch.cuda._sleep(CYCLES)
    earlier.fill_(255)
    filled = torch.cuda.Event()
    filled.record()
    del earlier
    op.workspace()
    assert filled.query()
    with torch.cuda.stream(side):
        op.backward(**inputs, grad_x=got)
    side.synchronize()
    assert torch.equal(got, want)


def test_captured_calls_leave_the_buffers_alone():
    """Calls captured on their own stream, replayed on another: as eager ones."""
    inputs = _distillation_inputs(64, 90)
    block, mlp = _block()
    op = TopKDistillation(64, 90, 4)
    mlp.workspace()
    want = torch.zeros(1, device="cuda"), torch.empty_like(block["x"])
    got = torch.zeros(1, device="cuda"), torch.empty_like(block["x"])

    def both(out):
        op.run(**inputs, loss_out=out[0])
        mlp.backward(**block, grad_x=out[1])

    both(want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        both(got)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph.replay()
        graph.replay()
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
