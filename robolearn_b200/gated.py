"""Host wrapper of the gated feed-forward block (``rl2_gated_*``): ``h = act(x Wg^T) * (x Wu^T)``
and its backward pass on the tcgen05 tensor cores, without storing either projection."""

from __future__ import annotations

import ctypes

import torch

from . import _native as N

DTYPES = {torch.float16: 0, torch.bfloat16: 1}
ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}


def _matrix(name: str, t: torch.Tensor, rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """Refuse what the kernels cannot read: shape, type, device, row layout."""
    if t.shape != (rows, cols):
        raise ValueError(f"{name} must have shape ({rows}, {cols}), got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")
    if cols > 1 and t.stride(1) != 1:
        raise ValueError(f"{name} must have contiguous rows (column stride 1, got {t.stride(1)})")
    return t


def _ld(t: torch.Tensor) -> int:
    """Row stride in elements; a single row's is free, so it is its padded length (16-byte multiples)."""
    if t.shape[0] > 1:
        return t.stride(0)
    quantum = 16 // t.element_size()
    return -(-t.shape[1] // quantum) * quantum


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
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self._lib = N.load()
        desc = N.GatedDesc(rows=self.rows, features=self.features, hidden=self.hidden, dtype=DTYPES[dtype],
                           activation=ACTIVATIONS[activation])
        with torch.cuda.device(self.device):
            self.handle = N.created(self._lib.rl2_gated_create(ctypes.byref(desc)), "create gated MLP plan")
        self._workspace = None

    def workspace_bytes(self) -> int:
        return self._lib.rl2_gated_workspace_bytes(self.handle)

    def workspace(self) -> torch.Tensor:
        """The backward's workspace (allocate it here before capturing a CUDA graph)."""
        if self._workspace is None:
            self._workspace = torch.empty(self.workspace_bytes(), dtype=torch.uint8, device=self.device)
        return self._workspace

    def forward(self, *, x, gate_weight, up_weight, out, health=None, stream=None) -> None:
        """``out = act(x gate_weight^T) * (x up_weight^T)`` for ``x.shape[0]`` <= ``rows`` rows."""
        rows, K, F, dt, dev = x.shape[0], self.features, self.hidden, self.dtype, self.device
        _matrix("x", x, rows, K, dt, dev)
        _matrix("gate_weight", gate_weight, F, K, dt, dev)
        _matrix("up_weight", up_weight, F, K, dt, dev)
        _matrix("out", out, rows, F, dt, dev)
        a = N.GatedForwardArgs(rows, x.data_ptr(), _ld(x), gate_weight.data_ptr(), _ld(gate_weight),
                               up_weight.data_ptr(), _ld(up_weight), out.data_ptr(), _ld(out), N.ptr(health))
        N.check(self._lib.rl2_gated_forward(self.handle, ctypes.byref(a), N.raw_stream(stream, self.device.index)), "gated MLP forward")

    def backward(self, *, x, gate_weight, up_weight, grad_out, grad_x=None, grad_gate=None, grad_up=None,
                 grad_weight_scale=None, health=None, stream=None) -> None:
        """Gradients of ``sum(out * grad_out)``: ``grad_x`` (optional) in the operand type, ``grad_gate`` and
        ``grad_up`` (both or neither) in the operand type or both fp32, times ``grad_weight_scale`` (one device
        float, optional: the inverse loss scale). They are assigned."""
        rows, K, F, dt, dev = x.shape[0], self.features, self.hidden, self.dtype, self.device
        _matrix("x", x, rows, K, dt, dev)
        _matrix("gate_weight", gate_weight, F, K, dt, dev)
        _matrix("up_weight", up_weight, F, K, dt, dev)
        _matrix("grad_out", grad_out, rows, F, dt, dev)
        if (grad_gate is None) != (grad_up is None):
            raise ValueError("grad_gate and grad_up come together")
        a = N.GatedBackwardArgs(rows=rows, x=x.data_ptr(), ldx=_ld(x), gate_weight=gate_weight.data_ptr(),
                                ld_gate=_ld(gate_weight), up_weight=up_weight.data_ptr(), ld_up=_ld(up_weight),
                                grad_out=grad_out.data_ptr(), ld_grad_out=_ld(grad_out), health=N.ptr(health),
                                workspace=self.workspace().data_ptr())
        if grad_x is not None:
            _matrix("grad_x", grad_x, rows, K, dt, dev)
            a.grad_x, a.ld_grad_x = grad_x.data_ptr(), _ld(grad_x)
        if grad_gate is not None:
            wt = grad_gate.dtype
            if wt not in (dt, torch.float32):
                raise ValueError(f"weight gradients must be {dt} or float32, got {wt}")
            _matrix("grad_gate", grad_gate, F, K, wt, dev)
            _matrix("grad_up", grad_up, F, K, wt, dev)
            a.grad_gate, a.ld_grad_gate = grad_gate.data_ptr(), _ld(grad_gate)
            a.grad_up, a.ld_grad_up = grad_up.data_ptr(), _ld(grad_up)
            a.grad_weight_fp32 = int(wt == torch.float32)
            if grad_weight_scale is not None:
                if grad_weight_scale.numel() != 1 or grad_weight_scale.dtype != torch.float32 or grad_weight_scale.device != dev:
                    raise ValueError(f"grad_weight_scale must be one float32 on {dev}")
                a.grad_weight_scale = grad_weight_scale.data_ptr()
        N.check(self._lib.rl2_gated_backward(self.handle, ctypes.byref(a), N.raw_stream(stream, self.device.index)), "gated MLP backward")

    def close(self) -> None:
        if self.handle:
            self._lib.rl2_gated_destroy(self.handle)
            self.handle = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
