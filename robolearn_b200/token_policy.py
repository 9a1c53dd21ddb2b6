"""A policy over discrete tokens (binned actions, skills), distilled from a teacher: the gated block,
the distillation objective and the sampler together with the dense products and the optimizer.

    h0     = obs W_in^T
    h1     = h0 + (act(h0 W_gate^T) * (h0 W_up^T)) W_down^T
    logits = h1 W_head^T

fp16 operands, fp32 sums, master weights, logits and Adam; gradients carry the optimizer's dynamic loss
scale. ``TokenPolicy.act`` draws tokens, ``TokenPolicy.distill_update`` makes one step towards a teacher's
top logits. Both only launch kernels on fixed buffers. ``python -m robolearn_b200.token_policy`` distills
a small policy from a fixed random one and prints how the loss falls.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _native as N
from .dense import FP16, TF32X3, DensePlan, operand_ld
from .distillation import TopKDistillation
from .gated import GatedMLP
from .token_sampling import TokenSampler

_STATE_FLOATS = 9  # rl2_adam_prepare's optimizer state


class _Weight:
    """One weight matrix: fp32 parameters and gradient in the arenas (rows padded to 16 bytes where ``aligned``, as the gated
    block writes them), fp16 operand plane with padded rows."""

    def __init__(self, out: int, inp: int, offset: int, plane_offset: int, aligned: bool):
        self.out, self.inp, self.offset, self.plane_offset, self.ld = out, inp, offset, plane_offset, operand_ld(inp, FP16)
        self.arena_ld = operand_ld(inp, TF32X3) if aligned else inp

    def arena(self, flat: torch.Tensor) -> torch.Tensor:
        return flat[self.offset:self.offset + self.out * self.arena_ld].view(self.out, self.arena_ld)[:, :self.inp]

    def plane(self, flat: torch.Tensor) -> torch.Tensor:
        return flat[self.plane_offset:self.plane_offset + self.out * self.ld].view(self.out, self.ld)[:, :self.inp]


class TokenPolicy:
    """Fixed batch of ``rows`` observations; ``top`` teacher entries a row in ``distill_update``."""

    def __init__(self, observation_dim: int, tokens: int, rows: int, *, hidden: int = 512, expand: int = 4, top: int = 8,
                 activation: str = "silu", learning_rate: float = 3e-4, seed: int = 0, device="cuda"):
        dev = torch.device(device)
        self.rows, self.tokens, self.hidden = rows, tokens, hidden
        wide = hidden * expand
        lib = self._lib = N.load()
        # ---- parameters: in, gate, up, down, head
        offset = plane = 0
        self.weights: dict[str, _Weight] = {}
        for name, out, inp in (("in", hidden, observation_dim), ("gate", wide, hidden), ("up", wide, hidden),
                               ("down", hidden, wide), ("head", tokens, hidden)):
            self.weights[name] = w = _Weight(out, inp, offset, plane, name in ("gate", "up"))
            offset += -(-out * w.arena_ld // 4) * 4
            plane += out * w.ld
        gen = torch.Generator().manual_seed(seed)
        host = torch.zeros(offset)
        for w in self.weights.values():
            w.arena(host).copy_(torch.randn(w.out, w.inp, generator=gen) / math.sqrt(w.inp))
        self.params = host.to(dev)
        f32 = dict(dtype=torch.float32, device=dev)
        self.grads, self.m1, self.m2 = (torch.zeros(offset, **f32) for _ in range(3))
        self.planes = torch.zeros(plane, dtype=torch.float16, device=dev)
        self.scale, self.inverse_scale = torch.full((1,), 65536.0, **f32), torch.full((1,), 1 / 65536.0, **f32)
        self.found_inf = torch.zeros(1, dtype=torch.int32, device=dev)
        self.health = torch.zeros(1, dtype=torch.int32, device=dev)
        self.opt_state = torch.zeros(_STATE_FLOATS, **f32)
        self.opt_state[6] = 65536.0
        segments = [(w.offset + r * w.arena_ld, -1, w.plane_offset + r * w.ld, w.inp, 0)
                    for w in self.weights.values() for r in range(w.out)]
        self._segments, self._count, self._warp_segments = N.segment_table(segments, dev)
        # ---- buffers
        def half(cols):
            return torch.zeros(rows, operand_ld(cols, FP16), dtype=torch.float16, device=dev)

        self.observation_dim, self.wide = observation_dim, wide
        self.obs, self._h0, self._h1, self._gated = half(observation_dim), half(hidden), half(hidden), half(wide)
        self._dh1, self._dgated, self._dx = half(hidden), half(wide), half(hidden)
        self._residual = torch.zeros(rows, hidden, **f32)
        self.logits = torch.zeros(rows, operand_ld(tokens, FP16), **f32)
        self._dlogits = half(tokens)
        self.loss, self.row_loss = torch.zeros(1, **f32), torch.zeros(rows, **f32)
        self.actions = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.log_probs = torch.zeros(rows, **f32)
        # ---- operators and products
        self.gated = GatedMLP(rows, hidden, wide, dtype=torch.float16, activation=activation, device=dev)
        self.gated.workspace()
        self.objective = TopKDistillation(rows, tokens, top, device=dev)
        self.sampler = TokenSampler(rows, tokens, device=dev)
        self._forward = [self._product("in", self.obs, d=self._residual, out=self._h0), self._run_gated,
                         self._product("down", self._gated, residual=self._residual, out=self._h1),
                         self._product("head", self._h1, d=self.logits)]
        self._backward = [self._weight_gradient("head", self._dlogits, self._h1),
                          self._input_gradient("head", self._dlogits, self._dh1),
                          self._weight_gradient("down", self._dh1, self._gated),
                          self._input_gradient("down", self._dh1, self._dgated), self._run_gated_backward,
                          self._weight_gradient("in", self._dx, self.obs),
                          self._weight_gradient("in", self._dh1, self.obs, accumulate=True)]
        self._optimizer = self._adam(learning_rate)
        self.refresh_planes()

    # ------------------------------------------------------------------ launches
    def _weight_plane(self):
        return N.Plane(h16=self.planes.data_ptr())

    def _operand_plane(self, t):
        return N.Plane(h16=t.data_ptr(), ld=t.stride(0), found_inf=self.found_inf.data_ptr())

    def _product(self, name, x, d=None, residual=None, out=None) -> DensePlan:
        """``x W^T (+ residual)`` as fp32 (``d``) and / or an fp16 operand (``out``)."""
        w = self.weights[name]
        plane = None if out is None else N.Plane(h16=out.data_ptr(), ld=out.stride(0))
        return DensePlan(kind=FP16, m=self.rows, n=w.out, k=w.inp, a=x, lda=x.stride(0), b=w.plane(self.planes), ldb=w.ld, d=d,
                         ldd=0 if d is None else d.stride(0), residual=residual,
                         ldr=0 if residual is None else residual.stride(0), out_plane=plane, health=self.health)

    def _input_gradient(self, name, dy, dx) -> DensePlan:
        """``dx = dy W``, an operand of the next products (its overflow skips the step)."""
        w = self.weights[name]
        return DensePlan(kind=FP16, m=self.rows, n=w.inp, k=w.out, a=dy, lda=dy.stride(0), b=w.plane(self.planes), ldb=w.ld,
                         b_major=1, d=None, ldd=0, out_plane=self._operand_plane(dx), health=self.health)

    def _weight_gradient(self, name, dy, x, accumulate=False) -> DensePlan:
        """``dW (+)= dy^T x / loss scale``."""
        w = self.weights[name]
        return DensePlan(kind=FP16, m=w.out, n=w.inp, k=self.rows, a=dy, lda=dy.stride(0), a_major=1, b=x, ldb=x.stride(0),
                         b_major=1, d=w.arena(self.grads), ldd=w.arena_ld, accumulate=accumulate, scale=self.inverse_scale,
                         health=self.health)

    def _gated_weights(self):
        return dict(gate_weight=self.weights["gate"].plane(self.planes), up_weight=self.weights["up"].plane(self.planes))

    def _run_gated(self):
        self.gated.forward(x=self._h0[:, :self.hidden], out=self._gated[:, :self.wide], health=self.health, **self._gated_weights())

    def _run_gated_backward(self):
        self.gated.backward(x=self._h0[:, :self.hidden], grad_out=self._dgated[:, :self.wide], grad_x=self._dx[:, :self.hidden],
                            grad_gate=self.weights["gate"].arena(self.grads), grad_up=self.weights["up"].arena(self.grads),
                            grad_weight_scale=self.inverse_scale, found_inf=self.found_inf, health=self.health,
                            **self._gated_weights())

    def _adam(self, learning_rate: float):
        prepare = N.AdamPrepareArgs(state=self.opt_state.data_ptr(), found_inf=self.found_inf.data_ptr(), formula=0, beta1=0.9,
                                    beta2=0.999, lr_init=learning_rate, lr_peak=learning_rate, lr_end=learning_rate,
                                    warmup_steps=0.0, decay_steps=1.0, scaler=1, growth=2.0, backoff=0.5,
                                    growth_interval=2000, scale_out=self.scale.data_ptr(),
                                    inv_scale_out=self.inverse_scale.data_ptr())
        step = self._adam_args(self.grads, self.opt_state)

        def run():
            s = N.stream_ptr()
            N.check(self._lib.rl2_adam_prepare(ctypes.byref(prepare), s), "token policy Adam prepare")
            N.check(self._lib.rl2_adam_step(ctypes.byref(step), s), "token policy Adam step")

        return run

    def _adam_args(self, grads, state):
        return N.AdamArgs(params=self.params.data_ptr(), grads=N.ptr(grads), m=self.m1.data_ptr(), v=self.m2.data_ptr(),
                          segments=self._segments.data_ptr(), count=self._count, state=N.ptr(state), formula=0, beta1=0.9,
                          beta2=0.999, eps=1e-8, project=0, weight_plane=self._weight_plane(), target_params=None, tau=0.0,
                          target_plane=N.Plane(), warp_segments=self._warp_segments)

    def refresh_planes(self) -> None:
        """Rewrite the fp16 weight planes from the fp32 parameters (after setting parameters by hand)."""
        N.check(self._lib.rl2_adam_step(ctypes.byref(self._adam_args(None, None)), N.stream_ptr()), "refresh weight planes")

    # ------------------------------------------------------------------ the policy
    def load_observations(self, obs: torch.Tensor) -> None:
        """The batch's observations [rows, observation_dim] (or one for all rows)."""
        if obs.shape not in ((self.rows, self.observation_dim), (1, self.observation_dim)):
            raise ValueError(f"observations must be of shape ({self.rows}, {self.observation_dim}), got {tuple(obs.shape)}")
        self.obs[:, :self.observation_dim].copy_(obs)

    def forward(self) -> torch.Tensor:
        """Logits [rows, tokens] (fp32) of the loaded observations."""
        for launch in self._forward:
            launch()
        return self.logits[:, :self.tokens]

    def act(self, obs: torch.Tensor, uniforms: torch.Tensor, **filters) -> tuple[torch.Tensor, torch.Tensor]:
        """One token per observation and its log-probability among the tokens kept (``temperature``, ``top_k``,
        ``top_p``, ``min_p``), from given uniforms."""
        self.load_observations(obs)
        self.sampler.run(logits=self.forward(), uniforms=uniforms, tokens=self.actions, log_probs=self.log_probs,
                         health=self.health, **filters)
        return self.actions, self.log_probs

    def gradients(self, teacher_values, teacher_indices, temperature: float = 1.0, row_weight=None) -> None:
        """Forward, objective and backward of the loaded observations: ``loss`` (mean over rows) and ``grads``."""
        logits = self.forward()
        self.objective.run(logits=logits, teacher_values=teacher_values, teacher_indices=teacher_indices,
                           temperature=temperature, row_weight=row_weight, loss_weight=1.0 / self.rows,
                           row_loss=self.row_loss, loss_out=self.loss, dlogits=self._dlogits[:, :self.tokens],
                           grad_scale=self.scale, health=self.health)
        for launch in self._backward:
            launch()

    def distill_update(self, obs, teacher_values, teacher_indices, temperature: float = 1.0, row_weight=None) -> torch.Tensor:
        """One step towards the teacher; the loss before it (device tensor)."""
        self.load_observations(obs)
        self.gradients(teacher_values, teacher_indices, temperature, row_weight)
        self._optimizer()
        return self.loss


def main(steps: int = 400) -> None:
    rows, obs_dim, tokens, top = 1024, 64, 256, 16
    teacher = TokenPolicy(obs_dim, tokens, rows, hidden=256, seed=1)
    student = TokenPolicy(obs_dim, tokens, rows, hidden=128, seed=2, top=top, learning_rate=1e-3)
    gen = torch.Generator(device="cuda").manual_seed(0)
    for step in range(steps + 1):
        obs = torch.randn(rows, obs_dim, generator=gen, device="cuda")
        teacher.load_observations(obs)
        values, indices = torch.topk(teacher.forward() * 3.0, top, dim=1)
        loss = student.distill_update(obs, values, indices)
        if step % 100 == 0:
            print(f"step {step}: loss {loss.item():.4f}")
    uniforms = torch.rand(rows, generator=gen, device="cuda")
    drawn, log_probs = student.act(obs, uniforms, temperature=0.8, top_k=top, top_p=0.95)
    hits = (drawn[:, None] == indices).any(1).float().mean().item()
    print(f"drawn tokens among the teacher's top {top}: {hits:.2f}, mean log-probability {log_probs.mean().item():.2f}")


if __name__ == "__main__":
    main()
