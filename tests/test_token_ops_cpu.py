"""Distillation and token sampling without a GPU: the C entries refuse bad arguments before any device
work, with a message."""

import ctypes
import math

import pytest

from robolearn_b200 import _native as N

FAKE = 0x1000


def _error():
    return N.load().rl2_last_error().decode()


def distill(**change):
    good = dict(rows=4, vocab=50, top=3, logits=FAKE, ld_logits=50, teacher_values=FAKE, ld_values=3,
                teacher_indices=FAKE, ld_indices=3, index_bits=64, temperature=1.0, loss_weight=1.0, row_loss=FAKE,
                dlogits=2 * FAKE, ld_dlogits=50, counter=FAKE)
    return N.load().rl2_distill_topk(ctypes.byref(N.DistillArgs(**{**good, **change})), None)


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows >= 0"), (dict(vocab=0), "vocab >= 1"), (dict(top=0), "teacher entries"),
    (dict(top=1025), "teacher entries"), (dict(logits_dtype=3), "types are"), (dict(values_dtype=-1), "types are"),
    (dict(dlogits_dtype=7), "types are"), (dict(index_bits=16), "32 or 64"), (dict(temperature=0.0), "temperature"),
    (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature"),
    (dict(loss_out=FAKE, counter=None), "counter"), (dict(logits=None), "non-null"), (dict(row_loss=None), "non-null"),
    (dict(teacher_values=None), "non-null"), (dict(teacher_indices=None), "non-null"), (dict(ld_logits=49), "shorter"),
    (dict(ld_values=2), "shorter"), (dict(ld_indices=0), "shorter"), (dict(ld_dlogits=49), "shorter"),
    (dict(logits=FAKE + 2), "aligned"), (dict(teacher_indices=FAKE + 4), "aligned"), (dict(dlogits=FAKE), "overwrite"),
])
def test_distillation_refuses(change, message):
    assert distill(**change) == -1 and message in _error()


def sample(**change):
    good = dict(rows=4, vocab=50, logits=FAKE, ld_logits=50, uniforms=FAKE, temperature=1.0, top_p=1.0, tokens=FAKE)
    return N.load().rl2_sample_tokens(ctypes.byref(N.SampleArgs(**{**good, **change})), None)


@pytest.mark.parametrize("change,message", [
    (dict(rows=-1), "rows >= 0"), (dict(vocab=0), "tokens are needed"), (dict(vocab=(1 << 20) + 1), "tokens are needed"),
    (dict(logits_dtype=3), "types are"), (dict(temperature=-1.0), "temperature >= 0"),
    (dict(temperature=math.nan), "temperature >= 0"), (dict(top_p=math.nan), "top_p"), (dict(min_p=1.5), "min_p"),
    (dict(min_p=math.nan), "min_p"), (dict(logits=None), "non-null"), (dict(uniforms=None), "non-null"),
    (dict(tokens=None), "non-null"), (dict(ld_logits=49), "shorter"), (dict(logits=FAKE + 1), "aligned"),
])
def test_sampling_refuses(change, message):
    assert sample(**change) == -1 and message in _error()


def test_null_arguments_and_no_rows():
    lib = N.load()
    assert lib.rl2_distill_topk(None, None) == -1 and "null" in _error()
    assert lib.rl2_sample_tokens(None, None) == -1 and "null" in _error()
    assert distill(rows=0) == 0 and sample(rows=0) == 0
