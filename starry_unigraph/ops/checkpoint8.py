"""Activations kept in 8 bits between the forward and the backward pass.

Format: groups of 32 neighbouring values of a row share one fp32 scale,
``scale = amax / 127`` and ``code = rint(v * (127 / amax))`` (the division and the
product by 1/127 each rounded once), 1.125 bytes a value. Rounding moves a value by at
most half a scale. A group whose largest magnitude is below 2^-100 reads back as
zeros; a group that holds a NaN or an infinity has the scale NaN and reads back as NaN,
so that a broken activation shows in the gradients.

* ``quantize8(x)`` -> ``Packed8``; ``Packed8.dequantize(dtype=None)`` back to x's type.
* ``with saved8(): loss = model(...)``: every activation that an autograd node of the
  block saves is kept in 8 bits (the framework's own ops and torch's alike) and restored
  when its backward pass asks for it. Parameters, integer tensors and small tensors stay
  as they are. A saved ReLU output below half its group's
  scale reads back as zero and passes no gradient.
* ``gated_scan`` and ``norm_residual`` take ``checkpoint="int8"``: their own kernels write
  the codes while they read the inputs and read the codes in the backward pass, with no
  restored copy in between.

On CPU tensors the same functions run the same arithmetic with torch operations.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from starry_unigraph.ops import cuda_ext

GROUP = 32


def check_checkpoint(value: str | None) -> bool:
    """True for ``"int8"``, False for None."""
    if value not in (None, "int8"):
        raise ValueError(f'checkpoint must be None or "int8", got {value!r}')
    return value == "int8"


def check_positive(value: float, name: str, dtype: torch.dtype) -> float:
    """A rate or eps as a float: positive and finite once rounded to the type that the formulas run in."""
    value = float(value)
    least, most = (0.0, float("inf")) if dtype == torch.float64 else (2.0 ** -150, 2.0 ** 128 - 2.0 ** 103)
    if not least < value < most:
        raise ValueError(f"{name} must be positive and finite, got {value}")
    return value


def _quantize_torch(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of [rows, H] with torch operations (fp32; fp64 inputs stay fp64)."""
    v = x if x.dtype == torch.float64 else x.float()
    v = F.pad(v, (0, -x.size(1) % GROUP)).unflatten(1, (-1, GROUP))
    top = v.abs().amax(2, keepdim=True)
    tiny, bad = top < 2.0 ** -100, ~torch.isfinite(top)
    zero = torch.zeros_like(top)
    inv = torch.where(tiny | bad, zero, torch.full_like(top, 127.0) / top)
    scale = torch.where(tiny, zero, torch.where(bad, torch.full_like(top, float("nan")), top * (1.0 / 127.0)))
    codes = torch.nan_to_num(torch.round(v * inv), nan=0.0)
    return codes.flatten(1)[:, : x.size(1)].to(torch.int8).contiguous(), scale.squeeze(2)


def _dequantize_torch(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    wide = scales.repeat_interleave(GROUP, dim=1)[:, : codes.size(1)]
    return (codes.to(wide.dtype) * wide).to(dtype)


_BITS = {2: torch.int16, 4: torch.int32, 8: torch.int64}


def _hidden(t: torch.Tensor | None) -> torch.Tensor | None:
    """The bits of t as integers, which saved-tensor hooks leave alone (the values of codes and kept
    states must not be packed again); back by ``view(dtype)``."""
    return None if t is None else t.view(_BITS[t.element_size()])


def _shown(t: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor | None:
    return None if t is None else t.view(dtype)


@dataclass
class Packed8:
    """8-bit codes [rows, H] and scales [rows, ceil(H / 32)] of a tensor of `shape` and `dtype`."""

    codes: torch.Tensor
    scales: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel() * self.scales.element_size()

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        dtype = self.dtype if dtype is None else dtype
        if self.codes.is_cuda:
            if dtype not in (torch.float32, torch.bfloat16):
                raise ValueError(f"dequantize: float32 or bfloat16 on CUDA, got {dtype}")
            out = cuda_ext().dequantize8(self.codes, self.scales, dtype == torch.bfloat16)
        else:
            out = _dequantize_torch(self.codes, self.scales, dtype)
        return out if out.shape == self.shape else out.view(self.shape)


def quantize8(x: torch.Tensor) -> Packed8:
    """8-bit codes of x along its last dimension (float32 or bfloat16; on CPU float64 too)."""
    if x.is_cuda:
        codes, scales = cuda_ext().quantize8(x)
        return Packed8(codes, scales, x.shape, x.dtype)
    if x.dim() == 0 or x.size(-1) == 0:
        raise ValueError("quantize8: x needs a last dimension of at least one value")
    if not x.is_floating_point():
        raise ValueError(f"quantize8: a floating tensor is wanted, got {x.dtype}")
    rows = x.detach().reshape(-1, x.size(-1))
    if rows.size(1) > 1 and rows.stride(1) != 1:
        rows = rows.contiguous()
    codes, scales = _quantize_torch(rows)
    return Packed8(codes, scales, x.shape, x.dtype)


@contextmanager
def saved8(min_numel: int = 1 << 16):
    """Keep the activations that autograd saves inside the block in 8 bits: dense float32
    and bfloat16 tensors of at least two dimensions and `min_numel` values that are neither
    parameters (``nn.Parameter``, frozen or not, or another leaf that requires a gradient) nor
    views of one, as the transposed weight that torch's linear saves. The recurrence's kept
    states and the scales of codes stay exact. A tensor that several nodes save is packed for
    each of them."""

    def pack(t: torch.Tensor):
        if (t.layout != torch.strided or t.dtype not in (torch.float32, torch.bfloat16) or t.dim() < 2
                or t.numel() < max(1, min_numel)):
            return t
        owner = t if t._base is None else t._base
        if isinstance(owner, torch.nn.Parameter) or (owner.is_leaf and owner.requires_grad):
            return t
        return quantize8(t)

    def unpack(p):
        return p.dequantize() if isinstance(p, Packed8) else p

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        yield
