"""Host wrapper of the gated feed-forward block (``rl2_gated_*``): ``h = act(x Wg^T) * (x Wu^T)``
and its backward pass on the tcgen05 tensor cores, without storing either projection."""

from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _native as N

DTYPES = {torch.float16: 0, torch.bfloat16: 1}
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}


class GatedMLP:
    """Plan of one gated block for up to ``rows`` rows: ``x`` [rows, features], ``gate_weight`` and
    ``up_weight`` [hidden, features], output [rows, hidden], all ``dtype`` (fp16 or bf16).

    Rows may be padded (any row stride that is a multiple of 16 bytes: ``dense.operand_ld``), bases are
    16-byte aligned. Outputs are the caller's; the backward's workspace is allocated on its first use
    and kept. Not thread-safe, and one call at a time per plan (the workspace is shared)."""

    def __init__(self, rows: int, features: int, hidden: int, *, dtype: torch.dtype = torch.float16,
                 activation: str = "silu", device="cuda"):
        if dtype not in DTYPES:
            raise ValueError(f"gated MLP operands are fp16 or bf16, got {dtype}")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
        self.handle = None
        self.rows, self.features, self.hidden = int(rows), int(features), int(hidden)
        self.dtype, self.activation = dtype, activation
        self._types = (dtype,)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._lib = N.load()
        desc = N.GatedDesc(rows=self.rows, features=self.features, hidden=self.hidden, dtype=DTYPES[dtype],
                           activation=ACTIVATIONS[activation])
        with contextlib.nullcontext() if self.device.index == torch.cuda.current_device() else torch.cuda.device(self.device):
            self.handle = N.created(self._lib.rl2_gated_create(ctypes.byref(desc)), "create gated MLP plan")
        self._workspace = None

    def _matrix(self, name, t, rows, cols, types=None) -> tuple[int, int]:
        address, ld = N.matrix(name, t, rows, cols, types or self._types, self.device)
        # a single row's stride is free: its length, padded to 16 bytes
        quantum = 8 if t.dtype != torch.float32 else 4
        return address, ld if rows > 1 else -(-cols // quantum) * quantum

    def workspace_bytes(self) -> int:
        return self._lib.rl2_gated_workspace_bytes(self.handle)

    def workspace(self) -> torch.Tensor:
        """The backward's workspace (allocate it here before capturing a CUDA graph)."""
        if self._workspace is None:
            self._workspace = torch.empty(self.workspace_bytes(), dtype=torch.uint8, device=self.device)
            self._buffers = N.Buffers(self.device, self._workspace)
        return self._workspace

    def forward(self, *, x, gate_weight, up_weight, out, health=None, stream=None) -> None:
        """``out = act(x gate_weight^T) * (x up_weight^T)`` for ``x.shape[0]`` <= ``rows`` rows."""
        rows, K, F = x.shape[0], self.features, self.hidden
        m = self._matrix
        a = N.GatedForwardArgs(rows, *m("x", x, rows, K), *m("gate_weight", gate_weight, F, K),
                               *m("up_weight", up_weight, F, K), *m("out", out, rows, F),
                               N.health_word(health, self.device))
        N.check(self._lib.rl2_gated_forward(self.handle, ctypes.byref(a), N.raw_stream(stream, self.device.index)),
                "gated MLP forward")

    def backward(self, *, x, gate_weight, up_weight, grad_out, grad_x=None, grad_gate=None, grad_up=None,
                 grad_weight_scale=None, found_inf=None, health=None, stream=None) -> None:
        """Gradients of ``sum(out * grad_out)``: ``grad_x`` (optional) in the operand type, ``grad_gate`` and
        ``grad_up`` (both or neither) in the operand type or both fp32, times ``grad_weight_scale`` (one device
        float, optional: the inverse loss scale). They are assigned. ``found_inf`` (one device int32, optional) becomes
        1 where one of them, or a hidden gradient on the way, overflows its type or is not a number."""
        rows, K, F = x.shape[0], self.features, self.hidden
        m = self._matrix
        if (grad_gate is None) != (grad_up is None):
            raise ValueError("grad_gate and grad_up come together")
        a = N.GatedBackwardArgs(rows, *m("x", x, rows, K), *m("gate_weight", gate_weight, F, K),
                                *m("up_weight", up_weight, F, K), *m("grad_out", grad_out, rows, F), health=N.health_word(health, self.device),
                                workspace=self.workspace().data_ptr())
        if grad_x is not None:
            a.grad_x, a.ld_grad_x = m("grad_x", grad_x, rows, K)
        if grad_gate is not None:
            types = (grad_gate.dtype,)
            if types[0] not in (self.dtype, torch.float32):
                raise ValueError(f"weight gradients must be {self.dtype} or float32, got {types[0]}")
            a.grad_gate, a.ld_grad_gate = m("grad_gate", grad_gate, F, K, types)
            a.grad_up, a.ld_grad_up = m("grad_up", grad_up, F, K, types)
            a.grad_weight_fp32 = int(types[0] == torch.float32)
            if grad_weight_scale is not None:
                a.grad_weight_scale = N.vector("grad_weight_scale", grad_weight_scale, 1, torch.float32, self.device)
        if found_inf is not None:
            a.found_inf = N.vector("found_inf", found_inf, 1, torch.int32, self.device)
        to = N.raw_stream(stream, self.device.index)
        self._buffers.use(to, stream)
        N.check(self._lib.rl2_gated_backward(self.handle, ctypes.byref(a), to), "gated MLP backward")

    def close(self) -> None:
        if self.handle:
            self._lib.rl2_gated_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
