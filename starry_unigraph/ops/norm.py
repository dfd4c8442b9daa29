"""Norms before and after a block, fused with the block's gate and residual scale.

    v = u / rms(u) * w_post          y = x + scale * sigmoid(gate) * v
    n = y / rms(y) * w_pre           rms(t) = sqrt(mean(t^2) + eps)

x is the residual stream, u the block's output, n the next block's input. One kernel reads
x, u and gate once and writes y and n; its backward pass reads x, u, gate and the two
gradients once. Statistics, sums and gradients of the vectors are fp32.

On CPU tensors the same functions run the formulas with torch operations.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from starry_unigraph.ops import cuda_ext
from starry_unigraph.ops.checkpoint8 import _hidden, _shown, check_checkpoint, check_positive, quantize8


def _norm_torch(x, u, gate, w_post, w_pre, scale, eps):
    dtype = x.dtype

    def wide(t):
        return t if t is None or t.dtype == torch.float64 else t.float()

    x, u, gate, w_post, w_pre, scale = (wide(t) for t in (x, u, gate, w_post, w_pre, scale))

    def rms(t, w):
        return t * torch.rsqrt(t.square().mean(-1, keepdim=True) + eps) * w

    y = x
    if u is not None:
        v = u if w_post is None else rms(u, w_post)
        if gate is not None:
            v = torch.sigmoid(gate) * v
        y = x + (v if scale is None else scale * v)
    return (None if u is None else y.to(dtype)), (None if w_pre is None else rms(y, w_pre).to(dtype))


class _NormCodes(torch.autograd.Function):
    """The CPU form of ``checkpoint="int8"``: outputs of the exact inputs, gradients at the codes' values."""

    @staticmethod
    def forward(ctx, x, u, gate, w_post, w_pre, scale, eps):
        wide = torch.float64 if x.dtype == torch.float64 else torch.float32
        held = [None if t is None else _hidden(quantize8(t).dequantize(wide)) for t in (x, u, gate)]
        ctx.save_for_backward(*held, w_post, w_pre, scale)
        ctx.meta = (eps, x.dtype, wide)
        ctx.set_materialize_grads(False)
        return _norm_torch(x, u, gate, w_post, w_pre, scale, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dn):
        eps, dtype, wide = ctx.meta
        saved = ctx.saved_tensors
        saved = (*(_shown(t, wide) for t in saved[:3]), *saved[3:])
        leaves = [None if t is None else t.detach().requires_grad_() for t in saved]
        with torch.enable_grad():
            outs = _norm_torch(*leaves, eps)
            pairs = [(o, g.to(o.dtype)) for o, g in zip(outs, (dy, dn)) if o is not None and g is not None]
            want = [t for t in leaves if t is not None]
            got = torch.autograd.grad([o for o, _ in pairs], want, [g for _, g in pairs], allow_unused=True)
        it = iter(got)
        grads = [None if t is None else next(it) for t in leaves]
        return (*[None if g is None else g.to(dtype) for g in grads[:3]], *grads[3:], None)


def norm_residual(x: torch.Tensor, u: torch.Tensor, w_post: torch.Tensor | None, w_pre: torch.Tensor | None = None, *,
                  gate: torch.Tensor | None = None, scale: torch.Tensor | None = None, eps: float = 1e-6,
                  checkpoint: str | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Returns ``(y, n)``; n is None without ``w_pre``.

    x, u, gate: ``[..., H]`` of one shape and type (float32 or bfloat16). w_post, w_pre, scale:
    ``[H]``, float32 or bfloat16. Without ``w_post`` u is added as it is, without ``gate`` or
    ``scale`` their factor is 1. H is at most 16384 on CUDA.

    checkpoint="int8" keeps x, u and gate in 8 bits (``quantize8``'s format) for the backward
    pass: gradients are those at the values of the codes, statistics recomputed from them."""
    return _call(x, u, gate, w_post, w_pre, scale, eps, checkpoint)


def rms_norm(x: torch.Tensor, w: torch.Tensor, *, eps: float = 1e-6, checkpoint: str | None = None) -> torch.Tensor:
    """``x / rms(x) * w``: the norm before the first block (types and checkpoint as above)."""
    return _call(x, None, None, None, w, None, eps, checkpoint)[1]


def _call(x, u, gate, w_post, w_pre, scale, eps, checkpoint):
    keep8 = check_checkpoint(checkpoint)
    if x.is_cuda:
        return cuda_ext().norm_residual(x, u, gate, w_post, w_pre, scale, eps, keep8)
    H = x.size(-1) if x.dim() else 0
    if H == 0:
        raise ValueError("norm_residual: x needs a last dimension of at least one value")
    eps = check_positive(eps, "norm_residual: eps", x.dtype)
    for name, t in (("u", u), ("gate", gate)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"norm_residual: {name} must have x's shape {tuple(x.shape)} and type {x.dtype}, got "
                             f"{tuple(t.shape)} {t.dtype}")
    for name, t in (("w_post", w_post), ("w_pre", w_pre), ("scale", scale)):
        if t is not None and tuple(t.shape) != (H,):
            raise ValueError(f"norm_residual: {name} must have shape ({H},), got {tuple(t.shape)}")
    args = (x, u, gate, w_post, w_pre, scale)
    if keep8 and torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        return _NormCodes.apply(*args, eps)
    return _norm_torch(*args, eps)
