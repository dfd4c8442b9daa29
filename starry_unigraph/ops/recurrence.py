"""Gated linear recurrence over node histories.

Per step and channel, from the input row ``p = (x | r | i)``, the channel's ``decay``
and the ``rate`` c:

    z = -c softplus(decay) sigmoid(r)     a = exp(z)
    h_t = a h_{t-1} + sqrt(1 - a^2) sigmoid(i) x

* ``gated_scan``: all steps of many sequences, with its backward pass. Sequences are
  ``[batch, steps, 3H]`` in any order of strides (a stack of snapshots transposed to
  node-major needs no copy), or histories of unequal length one after another,
  ``[rows, 3H]`` with ``offsets``. A masked step carries the state and does not read its
  input row.
* ``gated_scan_step``: one new token per row; reads and updates a table of fp32 states in
  place (no gradient).

The state is fp32 whatever the type of p. On CPU tensors the same functions run the
formulas with torch operations, step by step.
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from starry_unigraph.ops import cuda_ext
from starry_unigraph.ops.checkpoint8 import (_dequantize_torch, _hidden, _quantize_torch, _shown, check_checkpoint,
                                             check_positive)

STATE_EVERY = 16  # checkpoint="int8": steps between the fp32 states kept for the backward pass


def _scan_torch(p, decay, h0, mask, offsets, rate):
    """The recurrence step by step with torch operations (differentiable)."""
    wide = p if p.dtype == torch.float64 else p.float()
    dec = decay.to(wide.dtype)
    if offsets is not None:
        bounds = offsets.tolist()
        if not bounds or bounds[0] != 0 or bounds[-1] != p.size(0) or any(b < a for a, b in zip(bounds, bounds[1:])):
            raise ValueError("gated_scan: offsets must rise from 0 to the number of rows")
        outs, lasts = [], []
        for s, (a, b) in enumerate(zip(bounds, bounds[1:])):
            o, l = _scan_torch(wide[a:b].unsqueeze(0), dec, None if h0 is None else h0[s:s + 1],
                               None if mask is None else mask[a:b].unsqueeze(0), None, rate)
            outs.append(o[0])
            lasts.append(l)
        H = p.size(1) // 3
        h = torch.cat(outs) if outs else wide.new_zeros(0, H)
        return h.to(p.dtype), torch.cat(lasts) if lasts else wide.new_zeros(0, H)
    if mask is not None:
        wide = torch.where(mask.unsqueeze(-1), wide, torch.zeros_like(wide))
    x, r, i = wide.chunk(3, dim=-1)
    h = x.new_zeros(p.size(0), x.size(2)) if h0 is None else h0.to(wide.dtype)
    z = -rate * F.softplus(dec) * torch.sigmoid(r)
    a = torch.exp(z)
    open_ = z < 0  # a closed gate (a = 1) adds nothing; its root has no derivative
    add = torch.where(open_, torch.sqrt(-torch.expm1(2 * torch.where(open_, z, torch.full_like(z, -1.0)))),
                      torch.zeros_like(z)) * torch.sigmoid(i) * x
    outs = []
    for t in range(p.size(1)):
        if mask is None:
            h = a[:, t] * h + add[:, t]
        else:  # a step that does not count gives no gradient, whatever the state holds
            on = mask[:, t].unsqueeze(-1)
            h = torch.where(on, a[:, t] * torch.where(on, h, torch.zeros_like(h)) + add[:, t], h)
        outs.append(h)
    out = torch.stack(outs, 1) if outs else x
    return out.to(p.dtype), h


class _ThroughCodes(torch.autograd.Function):
    """The CPU form of ``checkpoint="int8"``: outputs of the exact inputs; gradients at the
    values of the codes, with the exact states before every STATE_EVERY-th step (packed:
    row of the packed axis)."""

    @staticmethod
    def forward(ctx, p, decay, h0, mask, offsets, rate):
        h, last = _scan_torch(p, decay, h0, mask, offsets, rate)
        wide = p if p.dtype == torch.float64 else p.float()
        if mask is not None:
            wide = torch.where(mask.unsqueeze(-1), wide, torch.zeros_like(wide))
        parts = wide.reshape(-1, p.size(-1) // 3)
        codes = _dequantize_torch(*_quantize_torch(parts), parts.dtype).view(wide.shape)
        full, _ = _scan_torch(wide, decay, h0, mask, offsets, rate)
        ctx.save_for_backward(_hidden(codes), _hidden(full), decay, _hidden(h0), mask, offsets)
        ctx.meta = (rate, p.dtype, codes.dtype, None if h0 is None else h0.dtype)
        return h, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dh, dlast):
        codes, full, decay, h0, mask, offsets = ctx.saved_tensors
        rate, dtype, wide, first_dtype = ctx.meta
        codes, full, h0 = _shown(codes, wide), _shown(full, wide), _shown(h0, first_dtype)
        E = dlast.to(codes.dtype)
        dp, ddecay = torch.zeros_like(codes), torch.zeros_like(decay, dtype=codes.dtype)
        dh0 = E.clone()
        packed = offsets is not None
        bounds = offsets.tolist() if packed else None
        runs = [(s, a, b) for s, (a, b) in enumerate(zip(bounds, bounds[1:]))] if packed else [(None, 0, codes.size(1))]
        for s, lo, hi in runs:
            e = E[s:s + 1] if packed else E
            at = (lambda v, a, b: v[a:b].unsqueeze(0)) if packed else (lambda v, a, b: v[:, a:b])
            start = lo
            cuts = [lo] + [t for t in range(lo + 1, hi) if t % STATE_EVERY == 0] + [hi]
            for a, b in reversed(list(zip(cuts, cuts[1:]))):
                if a == b:
                    continue
                first = (None if h0 is None else (h0[s:s + 1] if packed else h0)) if a == start else at(full, a - 1, a)[:, 0]
                with torch.enable_grad():
                    c = at(codes, a, b).detach().clone().requires_grad_()
                    d = decay.detach().to(codes.dtype).requires_grad_()
                    f = (c.new_zeros(c.size(0), c.size(2) // 3) if first is None else first.to(c.dtype)).detach().clone()
                    f.requires_grad_()
                    h, last = _scan_torch(c, d, f, None if mask is None else at(mask, a, b), None, rate)
                    gc, gd, e = torch.autograd.grad((h, last), (c, d, f), (at(dh, a, b).to(c.dtype), e))
                at(dp, a, b).copy_(gc)
                ddecay += gd
            if packed:
                dh0[s:s + 1] = e
            else:
                dh0 = e
        return (dp.to(dtype), ddecay.to(decay.dtype), dh0.to(h0.dtype) if h0 is not None else None, None, None, None)


def gated_scan(p: torch.Tensor, decay: torch.Tensor, h0: torch.Tensor | None = None, *,
               mask: torch.Tensor | None = None, offsets: torch.Tensor | None = None, rate: float = 8.0,
               checkpoint: str | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Runs the recurrence over every sequence; returns ``(h, last)``.

    p: ``[batch, steps, 3H]`` or, with ``offsets``, ``[rows, 3H]``; float32 or bfloat16.
    decay: ``[H]``, float32 or bfloat16. h0: ``[batch, H]`` first states (zeros when None).
    mask: bool ``[batch, steps]`` (packed ``[rows]``); a False step returns the state before
    it, reads nothing of p and gets no gradient. offsets: int64 ``[batch + 1]`` rising from 0
    to ``rows``; empty sequences return their first state. On CUDA, offsets that do not
    rise or leave the rows are reported by ``check_status()``; results are then undefined.
    h has p's type and layout; ``last`` is the fp32 state after each sequence.

    checkpoint="int8" keeps p in 8 bits (``quantize8``'s format, each of x, r and i in groups
    of its own) for the backward pass instead of p itself: gradients are those at the
    values of the codes, the states between fp32 ones that are kept every 16 steps (packed: rows of
    the packed axis) recomputed from them."""
    keep8 = check_checkpoint(checkpoint)
    if p.is_cuda:
        return cuda_ext().gated_scan(p, decay, h0, mask, offsets, rate, keep8)
    if p.dim() != (3 if offsets is None else 2) or p.size(-1) == 0 or p.size(-1) % 3:
        raise ValueError("gated_scan: p must be [batch, steps, 3H], or [rows, 3H] with offsets")
    rate = check_positive(rate, "gated_scan: rate", p.dtype)
    H = p.size(-1) // 3
    if tuple(decay.shape) != (H,):
        raise ValueError(f"gated_scan: decay must have shape ({H},), got {tuple(decay.shape)}")
    batch = p.size(0) if offsets is None else offsets.numel() - 1
    if h0 is not None and tuple(h0.shape) != (batch, H):
        raise ValueError(f"gated_scan: h0 must have shape ({batch}, {H}), got {tuple(h0.shape)}")
    if mask is not None and (mask.dtype != torch.bool or mask.shape != p.shape[:-1]):
        raise ValueError(f"gated_scan: mask must be bool of shape {tuple(p.shape[:-1])}")
    if keep8:
        return _ThroughCodes.apply(p, decay, h0, mask, offsets, rate)
    return _scan_torch(p, decay, h0, mask, offsets, rate)


def gated_scan_step(p: torch.Tensor, decay: torch.Tensor, state: torch.Tensor, rows: torch.Tensor | None = None, *,
                    rate: float = 8.0) -> torch.Tensor:
    """One step for each row of p ``[n, 3H]``; returns h ``[n, H]`` in p's type.

    state: fp32 table ``[table rows, H]``, updated in place: row ``rows[j]`` (int64, no row
    twice; None: row j) holds the state of row j. On CUDA a place outside the table is reported
    by ``check_status()``, its row of h is zero and nothing is written for it; on CPU it raises
    before anything is written. No gradient flows through a step."""
    if p.is_cuda:
        return cuda_ext().gated_scan_step(p, decay, state, rows, rate)
    if p.dim() != 2 or p.size(1) == 0 or p.size(1) % 3:
        raise ValueError("gated_scan_step: p must be [rows, 3H]")
    rate = check_positive(rate, "gated_scan_step: rate", p.dtype)
    if state.dtype not in (torch.float32, torch.float64) or state.dim() != 2 or state.size(1) * 3 != p.size(1):
        raise ValueError(f"gated_scan_step: state must be float32 [table rows, {p.size(1) // 3}]")
    if (state.size(0) if rows is None else rows.numel()) != p.size(0):
        raise ValueError("gated_scan_step: one place of the table per row of p is wanted")
    if tuple(decay.shape) != (state.size(1),):
        raise ValueError(f"gated_scan_step: decay must have shape ({state.size(1)},), got {tuple(decay.shape)}")
    if rows is not None:
        if rows.dtype not in (torch.int64, torch.int32) or rows.dim() != 1:
            raise ValueError("gated_scan_step: rows must be an int64 vector, one place per row of p")
        if rows.numel() and not 0 <= int(rows.min()) <= int(rows.max()) < state.size(0):
            raise IndexError(f"gated_scan_step: rows must be places of the table, 0 to {state.size(0) - 1}")
    with torch.no_grad():
        h, last = _scan_torch(p.unsqueeze(1), decay, state if rows is None else state[rows], None, None, rate)
        if rows is None:
            state.copy_(last)
        else:
            state[rows] = last.to(state.dtype)
        return h[:, 0]
