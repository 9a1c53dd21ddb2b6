"""The distillation refuses a gradient that shares memory with the logits, and nothing else, without a GPU: random pairs of
matrices against the bytes that they hold. A call whose matrices are apart is refused all the same, by a later check (a row
stride of the teacher's values), so none reaches a launch."""

import ctypes
import random

import pytest

from robolearn_b200 import _native as N

BASE = 0x100000
SIZE = [4, 2, 2]


def _refusal(rows, vocab, logits, ld_logits, kind, dlogits, ld_dlogits, grad_kind):
    args = N.DistillArgs(rows=rows, vocab=vocab, top=3, logits=logits, ld_logits=ld_logits, logits_dtype=kind, teacher_values=0x1000,
                         ld_values=2, teacher_indices=0x1000, ld_indices=3, index_bits=64, temperature=1.0, loss_weight=1.0,
                         row_loss=0x1000, dlogits=dlogits, ld_dlogits=ld_dlogits, dlogits_dtype=grad_kind)
    assert N.load().rl2_distill_topk(ctypes.byref(args), None) == -1
    return N.load().rl2_last_error().decode()


def _bytes(rows, vocab, base, ld, size):
    return {base + r * ld * size + b for r in range(rows) for b in range(vocab * size)}


@pytest.mark.parametrize("seed", range(6))
def test_overlap(seed):
    rng = random.Random(seed)
    seen = set()
    for _ in range(400):
        rows, vocab = rng.randint(1, 5), rng.randint(1, 6)
        kind, grad_kind = rng.randint(0, 2), rng.randint(0, 2)
        ld_a = vocab + rng.choice((0, 0, 1, vocab, 9))
        ld_b = ld_a * SIZE[kind] // SIZE[grad_kind] if rng.random() < 0.5 else vocab + rng.choice((0, 1, 7, 13))
        if ld_b < vocab:
            continue
        a, b = BASE, BASE + SIZE[grad_kind] * rng.randint(-60, 60)
        shared = bool(_bytes(rows, vocab, a, ld_a, SIZE[kind]) & _bytes(rows, vocab, b, ld_b, SIZE[grad_kind]))
        message = _refusal(rows, vocab, a, ld_a, kind, b, ld_b, grad_kind)
        assert ("may not overwrite" in message) == shared and ("shorter" in message) == (not shared), (rows, vocab, ld_a, ld_b, b - a)
        seen.add(shared)
    assert seen == {True, False}
