"""Host wrapper of the distillation objective from a teacher's top logits (``rl2_distill_topk``)."""

from __future__ import annotations

import ctypes

import torch

from . import _native as N

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_VOCAB = 1 << 30
INDEX_BITS = {torch.int32: 32, torch.int64: 64}


class TopKDistillation:
    """Persistent workspace of the objective for up to ``rows`` rows of ``vocab`` logits and ``top``
    teacher entries a row. One call at a time per object (the calls share its counter)."""

    def __init__(self, rows: int, vocab: int, top: int, device="cuda"):
        if rows < 1 or not 1 <= vocab <= MAX_VOCAB or not 1 <= top <= 1024:
            raise ValueError(f"rows and vocab (up to {MAX_VOCAB}) must be positive and top 1..1024, got {rows}, {vocab}, {top}")
        self.rows, self.vocab, self.top = int(rows), int(vocab), int(top)
        self._lib = N.load()
        self.counter = torch.zeros(1, dtype=torch.int32, device=device)
        self.row_loss = torch.zeros(self.rows, device=device)
        self.device = self.counter.device
        self._counter = self.counter.data_ptr()
        self._buffers = N.Buffers(self.device, self.counter, self.row_loss)

    def _matrix(self, name, t, rows, cols, types):
        return *N.matrix(name, t, rows, cols, types, self.device), types[t.dtype]

    def _vector(self, name, t, n):
        return N.vector(name, t, n, torch.float32, self.device)

    def run(self, *, logits, teacher_values, teacher_indices, temperature=1.0, row_weight=None, loss_weight=1.0,
            row_loss=None, loss_out=None, dlogits=None, grad_scale=None, health=None, stream=None) -> None:
        """Loss per row (``row_loss``, default ``self.row_loss``), total (``loss_out``) and the logits'
        gradient (``dlogits``, in its own type, times ``grad_scale``) for ``logits.shape[0]`` rows;
        formulas and special rows in include/rl2.h."""
        n = logits.shape[0]
        if n > self.rows:
            raise ValueError(f"at most {self.rows} rows, got {n}")
        a = N.DistillArgs(n, self.vocab, self.top, *self._matrix("logits", logits, n, self.vocab, DTYPES),
                          *self._matrix("teacher_values", teacher_values, n, self.top, DTYPES),
                          *self._matrix("teacher_indices", teacher_indices, n, self.top, INDEX_BITS), temperature, None,
                          loss_weight, counter=self._counter, health=N.health_word(health, self.device))
        if row_weight is not None:
            a.row_weight = self._vector("row_weight", row_weight, n)
        a.row_loss = self.row_loss.data_ptr() if row_loss is None else self._vector("row_loss", row_loss, n)
        if loss_out is not None:
            a.loss_out = self._vector("loss_out", loss_out, 1)
        if dlogits is not None:
            a.dlogits, a.ld_dlogits, a.dlogits_dtype = self._matrix("dlogits", dlogits, n, self.vocab, DTYPES)
        if grad_scale is not None:
            a.grad_scale = self._vector("grad_scale", grad_scale, 1)
        to = N.raw_stream(stream, self.device.index)
        self._buffers.use(to, stream)
        N.check(self._lib.rl2_distill_topk(ctypes.byref(a), to), "distillation objective")
