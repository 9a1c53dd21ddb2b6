"""Host wrapper of token sampling with temperature, top-k, top-p and min-p (``rl2_sample_tokens``)."""

from __future__ import annotations

import ctypes

import torch

from . import _native as N

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
MAX_VOCAB = 1 << 20


class TokenSampler:
    """Draws one token per row for up to ``rows`` rows of ``vocab`` logits. Holds no state: the random
    numbers are the caller's uniforms in [0, 1)."""

    def __init__(self, rows: int, vocab: int, device="cuda"):
        if rows < 1 or not 1 <= vocab <= MAX_VOCAB:
            raise ValueError(f"rows must be positive and vocab 1..{MAX_VOCAB}, got {rows}, {vocab}")
        self.rows, self.vocab = int(rows), int(vocab)
        self._lib = N.load()
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())

    def _vector(self, name, t, n, dtype=torch.float32):
        if t.shape != (n,) or t.dtype != dtype or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"{name} must be {n} contiguous {dtype} values on {self.device}")
        return t.data_ptr()

    def run(self, *, logits, uniforms, tokens, log_probs=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
            health=None, stream=None) -> None:
        """``tokens`` (int32) and ``log_probs`` (float32, optional) of ``logits.shape[0]`` rows. Each of
        ``temperature``, ``top_k``, ``top_p`` and ``min_p`` is one number for all rows or a device tensor
        with one value a row (float32; int32 for ``top_k``). Definition and special rows in include/rl2.h."""
        n = logits.shape[0]
        if n > self.rows or logits.shape != (n, self.vocab) or logits.dtype not in DTYPES or logits.device != self.device:
            raise ValueError(f"logits must be (up to {self.rows}, {self.vocab}) of fp32, fp16 or bf16 on {self.device}, "
                             f"got {tuple(logits.shape)} {logits.dtype} on {logits.device}")
        if self.vocab > 1 and logits.stride(1) != 1:
            raise ValueError("logits must have contiguous rows")
        a = N.SampleArgs(rows=n, vocab=self.vocab, logits=logits.data_ptr(),
                         ld_logits=logits.stride(0) if n > 1 else self.vocab, logits_dtype=DTYPES[logits.dtype],
                         uniforms=self._vector("uniforms", uniforms, n), top_p=1.0,
                         tokens=self._vector("tokens", tokens, n, torch.int32), health=N.ptr(health))
        if log_probs is not None:
            a.log_probs = self._vector("log_probs", log_probs, n)
        for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                                   ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
            if isinstance(value, torch.Tensor):
                setattr(a, name + "s", self._vector(name, value, n, dtype))
            else:
                setattr(a, name, value)
        N.check(self._lib.rl2_sample_tokens(ctypes.byref(a), N.raw_stream(stream, self.device.index)), "token sampling")
