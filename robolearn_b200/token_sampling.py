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

    def run(self, *, logits, uniforms, tokens, log_probs=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
            log_probs_of_logits=False, health=None, stream=None) -> None:
        """``tokens`` (int32) and ``log_probs`` (float32, optional) of ``logits.shape[0]`` rows. Each of
        ``temperature``, ``top_k``, ``top_p`` and ``min_p`` is one number for all rows or a device tensor
        with one value a row (float32; int32 for ``top_k``). ``log_probs`` are those of the draw, whose weights are
        multiples of 2^-30 of the best token's; ``log_probs_of_logits``: the logits' own among the tokens kept, for a learner
        that computes them again (they differ for tokens far below the best). Definition and special rows in include/rl2.h."""
        n, device = logits.shape[0], self.device
        if n > self.rows:
            raise ValueError(f"logits must be at most {self.rows} rows, got {n}")
        address, ld = N.matrix("logits", logits, n, self.vocab, DTYPES, device)
        a = N.SampleArgs(n, self.vocab, address, ld, DTYPES[logits.dtype], N.vector("uniforms", uniforms, n, torch.float32, device),
                         top_p=1.0, tokens=N.vector("tokens", tokens, n, torch.int32, device), health=N.health_word(health, device))
        if log_probs is not None:
            a.log_probs = N.vector("log_probs", log_probs, n, torch.float32, device)
            a.log_probs_of_logits = int(log_probs_of_logits)
        for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                                   ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
            if isinstance(value, torch.Tensor):
                setattr(a, name + "s", N.vector(name, value, n, dtype, device))
            else:
                setattr(a, name, value)
        N.check(self._lib.rl2_sample_tokens(ctypes.byref(a), N.raw_stream(stream, self.device.index)), "token sampling")
