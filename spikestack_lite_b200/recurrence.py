"""Training and streaming modules over the gated linear recurrence.

GatedRecurrence is a pre-norm temporal block for (T, B, N, d) planes: group
norm + SiLU per plane and sample, a projection to values and gates, the leaky
gated recurrence over the planes (ops.gated_recurrence), an output projection
and the residual with dropout.  Unlike the GSMC cell (nn/gsmc.py:96-148),
whose gates read the previous plane's spikes, its recurrence is linear in the
state: the planes are trained in parallel along time, and a stream is served
plane by plane with `step`.  No reference counterpart.
"""
import torch
import torch.nn as nn

from . import ops
from ._lib import EngineError
from .ops import engine_linear


class Dropout(nn.Module):
    """Counter-based dropout of a branch with its residual (ops.dropout).

    The key (seed, calls so far) is a device buffer advanced by every training
    call, also inside a captured graph, whose replays thus draw new masks; no
    mask is stored.  The buffer is not part of the state dict; manual_seed
    restarts it."""

    def __init__(self, p=0.1):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"dropout probability must lie in [0, 1], got {p}")
        self.p = float(p)
        seed = torch.randint(0, 1 << 62, (1,), dtype=torch.int64)
        self.register_buffer("key", torch.cat([seed, torch.zeros(1, dtype=torch.int64)]), persistent=False)

    def manual_seed(self, seed, calls=0):
        self.key.copy_(torch.tensor([int(seed), int(calls)], dtype=torch.int64))

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x
        key = self.key.clone()
        self.key[1:].add_(1)
        if residual is not None and x.dtype != residual.dtype:
            x = x.to(residual.dtype)
        return ops.dropout(x, self.p, key, residual=residual)

    def extra_repr(self):
        return f"p={self.p}"


def _linear(lin, x):
    """lin(x), at inference on the engine's fp32-accurate tensor-core linear."""
    y = engine_linear(lin, x) if x.dtype == torch.float32 else None
    return lin(x) if y is None else y


class GatedRecurrence(nn.Module):
    """x + dropout(W_o h) with h the leaky recurrence over dimension 0 of
    (v, g) = W_vg silu(group_norm(x)).  forward(x (T, B, N, d), state=None) ->
    (y, state); step(plane (B, N, d), state) -> (y, state) for one plane."""

    def __init__(self, d_model, groups=8, dropout=0.0, memory=(1.0, 6.0)):
        super().__init__()
        if d_model % groups:
            raise ValueError("d_model must be divisible by groups")
        self.d_model, self.groups = d_model, groups
        self.norm_weight = nn.Parameter(torch.ones(d_model))
        self.norm_bias = nn.Parameter(torch.zeros(d_model))
        self.eps = 1e-5
        self.vg_proj = nn.Linear(d_model, 2 * d_model)
        self.o_proj = nn.Linear(d_model, d_model)
        with torch.no_grad():  # gate biases: memories of a few planes to some hundred
            self.vg_proj.bias[d_model:].uniform_(*memory)
        self.dropout = Dropout(dropout) if dropout > 0.0 else None

    def _inputs(self, planes):
        """Values and gates (halves of one projection) of planes (P, N, d)."""
        u = ops.group_norm_act(planes, self.groups, self.norm_weight.float(), self.norm_bias.float(), self.eps,
                               act="silu")
        vg = _linear(self.vg_proj, u)
        return vg[..., :self.d_model], vg[..., self.d_model:]

    def _output(self, x, h):
        y = _linear(self.o_proj, h)
        return x + y if self.dropout is None else self.dropout(y, residual=x)

    def forward(self, x, state=None):
        if x.device.type != "cuda":
            raise EngineError("GatedRecurrence: CUDA input required (no CPU path)")
        if x.dim() != 4 or x.shape[-1] != self.d_model:
            raise EngineError(f"GatedRecurrence: x must be (T, B, N, {self.d_model}), got {tuple(x.shape)}")
        v, g = self._inputs(x.flatten(0, 1))
        h, state = ops.gated_recurrence(v.view(x.shape), g.view(x.shape), state, dim=0)
        return self._output(x, h), state

    @torch.no_grad()
    def step(self, plane, state=None):
        if plane.device.type != "cuda":
            raise EngineError("GatedRecurrence: CUDA input required (no CPU path)")
        if plane.dim() != 3 or plane.shape[-1] != self.d_model:
            raise EngineError(f"GatedRecurrence: plane must be (B, N, {self.d_model}), got {tuple(plane.shape)}")
        v, g = self._inputs(plane)
        if state is None:
            state = torch.zeros(plane.shape, dtype=torch.float32, device=plane.device)
        h, state = ops.gated_recurrence_step(v, g, state)
        return self._output(plane, h), state
