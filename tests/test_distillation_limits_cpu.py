"""Limits of the distillation without a GPU: vocabularies whose column indexes would leave 32 bits, temperatures whose
reciprocal leaves fp32. Every call is refused, by
the limit or by a later check (a row stride of the teacher's values), so none reaches a launch."""

import ctypes

import pytest

from robolearn_b200 import _native as N
from robolearn_b200.distillation import TopKDistillation


def _refusal(**change):
    good = dict(rows=1, vocab=50, top=3, logits=0x1000, ld_logits=1 << 32, teacher_values=0x1000, ld_values=2, teacher_indices=0x1000,
                ld_indices=3, index_bits=64, temperature=1.0, loss_weight=1.0, row_loss=0x1000)
    assert N.load().rl2_distill_topk(ctypes.byref(N.DistillArgs(**{**good, **change})), None) == -1
    return N.load().rl2_last_error().decode()


@pytest.mark.parametrize("vocab", [(1 << 30) + 1, (1 << 31) - 1100, (1 << 31) - 1])
def test_vocabulary(vocab):
    assert "2^30" in _refusal(vocab=vocab) and "shorter" in _refusal(vocab=1 << 30)
    with pytest.raises(ValueError, match="vocab"):
        TopKDistillation(1, vocab, 3)


@pytest.mark.parametrize("temperature", [1e-45, 1e-39, 4e-39])
def test_temperature(temperature):
    assert "reciprocal" in _refusal(temperature=temperature)
    for good in (4.3e-39, 1e-38, 1e-20, 1e30):
        assert "shorter" in _refusal(temperature=good)
