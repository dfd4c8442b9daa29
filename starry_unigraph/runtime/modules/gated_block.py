"""Stack of gated recurrent blocks over node histories.

Per layer, on rows of width H (one row per node and step):

    n = norm(y)                      p = W_p n + b_p,  g = W_g n + b_g
    h = gated_scan(p)                u = W_o h
    y <- y + scale * sigmoid(g) * norm(u)

The norm after a block, its gate and residual scale and the norm before the next block are
one kernel (``norm_residual``); the recurrence runs over all steps at once (``gated_scan``)
instead of one cell call per snapshot, and ``step`` advances every layer by one token on a
table of states. With ``checkpoint="int8"`` the recurrence and the norms keep their inputs
in 8 bits for the backward pass. Rows are taken in the type of the parameters (float32 or
bfloat16, on CPU float64 too); states are float32 (of float64 blocks float64).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from starry_unigraph.ops.checkpoint8 import check_checkpoint
from starry_unigraph.ops.dtdg import linear
from starry_unigraph.ops.norm import norm_residual, rms_norm
from starry_unigraph.ops.recurrence import gated_scan, gated_scan_step


class GatedRecurrentStack(nn.Module):
    def __init__(self, width: int, num_layers: int = 2, rate: float = 8.0, eps: float = 1e-6,
                 checkpoint: str | None = None) -> None:
        super().__init__()
        if width < 1 or num_layers < 1:
            raise ValueError("GatedRecurrentStack: width and num_layers must be positive")
        check_checkpoint(checkpoint)
        self.width, self.rate, self.eps, self.checkpoint = width, float(rate), float(eps), checkpoint
        self.proj = nn.ModuleList([nn.Linear(width, 3 * width) for _ in range(num_layers)])
        self.gate = nn.ModuleList([nn.Linear(width, width) for _ in range(num_layers)])
        self.out = nn.ModuleList([nn.Linear(width, width, bias=False) for _ in range(num_layers)])
        # decays of 0.9 to 0.999 a step at a half-open gate: softplus(decay) rate / 2 = -log(a)
        a = 1 - 10 ** -torch.linspace(1, 3, width)
        decay = torch.log(torch.expm1(-torch.log(a) * 2 / self.rate))
        self.decay = nn.ParameterList([nn.Parameter(decay.clone()) for _ in range(num_layers)])
        self.pre = nn.ParameterList([nn.Parameter(torch.ones(width)) for _ in range(num_layers + 1)])
        self.post = nn.ParameterList([nn.Parameter(torch.ones(width)) for _ in range(num_layers)])
        self.scale = nn.ParameterList([nn.Parameter(torch.full((width,), num_layers ** -0.5))
                                       for _ in range(num_layers)])

    @property
    def num_layers(self) -> int:
        return len(self.proj)

    def init_state(self, rows: int, device=None) -> list[torch.Tensor]:
        """Zero states, one table [rows, width] per layer."""
        device = self.decay[0].device if device is None else device
        dtype = torch.float64 if self.decay[0].dtype == torch.float64 else torch.float32
        return [torch.zeros(rows, self.width, device=device, dtype=dtype) for _ in range(self.num_layers)]

    def _layers(self, x, recur):
        """x [rows, width] through every layer; recur(layer, p) gives h."""
        x = x.to(self.pre[0].dtype)
        y, n = x, rms_norm(x, self.pre[0], eps=self.eps, checkpoint=self.checkpoint)
        for k in range(self.num_layers):
            p = linear(n, self.proj[k].weight, self.proj[k].bias)
            g = linear(n, self.gate[k].weight, self.gate[k].bias)
            u = linear(recur(k, p), self.out[k].weight)
            y, n = norm_residual(y, u, self.post[k], self.pre[k + 1], gate=g, scale=self.scale[k], eps=self.eps,
                                 checkpoint=self.checkpoint)
        return n

    def forward(self, x: torch.Tensor, state: list[torch.Tensor] | None = None, mask: torch.Tensor | None = None):
        """x [steps, rows, width] (snapshots stacked), state one [rows, width] per layer or
        None, mask bool [steps, rows]: False where a row is absent (its input is not read and
        its state stays). Returns (normed output [steps, rows, width], states)."""
        steps, rows, width = x.shape
        if width != self.width:
            raise ValueError(f"GatedRecurrentStack: rows of width {self.width} are wanted, got {width}")
        if mask is not None:  # NaN rows would reach the weight gradients
            x = torch.where(mask.unsqueeze(-1), x, torch.zeros_like(x))
        states: list[torch.Tensor] = []

        def recur(k, p):
            h, last = gated_scan(p.view(steps, rows, 3 * width).transpose(0, 1), self.decay[k],
                                 None if state is None else state[k], mask=None if mask is None else mask.t(),
                                 rate=self.rate, checkpoint=self.checkpoint)
            states.append(last)
            return h.transpose(0, 1).reshape(steps * rows, width)

        n = self._layers(x.reshape(steps * rows, width), recur)
        return n.view(steps, rows, width), states

    @torch.no_grad()
    def step(self, x: torch.Tensor, state: list[torch.Tensor], rows: torch.Tensor | None = None) -> torch.Tensor:
        """One new token x [n, width] per row; the layers' tables `state` advance in place at
        `rows` (every row when None). Returns the normed output [n, width]."""
        return self._layers(x, lambda k, p: gated_scan_step(p, self.decay[k], state[k], rows, rate=self.rate))
