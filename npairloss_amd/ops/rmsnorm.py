"""Root-mean-square norm over the last dimension, with the residual's addition
in front of it and an output in the input's type or in e4m3 with scales.

    s = x + residual                      (kept, in x's type)
    y = s / sqrt(mean(s^2) + eps) * weight

GPU tensors run the HIP kernels of csrc/rms_norm.hip (one pass over the rows
per direction); CPU tensors use the equivalent torch math.  Sums are fp32.
Rows have 1 to 16384 columns.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _backend

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_FP8 = torch.float8_e4m3fn
_FP8_MAX = 448.0
_TINY = 2.0 ** -126
MAX_COLUMNS = 16384


def _check(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor]):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_COLUMNS:
        raise ValueError(f"rms_norm: 1 to {MAX_COLUMNS} columns expected, got shape {tuple(x.shape)}")
    if x.dtype not in _FLOATS:
        raise TypeError(f"rms_norm: fp32, bf16 or fp16 expected, got {x.dtype}")
    if weight.shape != x.shape[-1:]:
        raise ValueError(f"rms_norm: weight {tuple(weight.shape)} does not fit rows of {x.shape[-1]}")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"rms_norm: weight is {weight.dtype}, x is {x.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"rms_norm: residual {tuple(residual.shape)} {residual.dtype} does not match "
                         f"x {tuple(x.shape)} {x.dtype}")
    for t in (weight, residual):
        if t is not None and t.device != x.device:
            raise ValueError(f"rms_norm: tensors on {x.device} and {t.device}")


class _RMSNormFn(torch.autograd.Function):
    """On the CPU; GPU tensors are recorded in csrc/autograd.cpp."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        ctx.has_residual = residual is not None
        s = x + residual if ctx.has_residual else x
        sf = s.float().contiguous()
        inv = torch.rsqrt(sf.square().mean(-1) + eps)
        y = (sf * inv.unsqueeze(-1) * weight.float()).to(x.dtype)
        ctx.save_for_backward(s, weight, inv)
        ctx.set_materialize_grads(False)
        return (y, s) if ctx.has_residual else y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dsum=None):
        s, weight, inv = ctx.saved_tensors
        if dy is None:  # only the sum was used
            return dsum, None, dsum, None
        n, g = s.float() * inv.unsqueeze(-1), dy.float()
        dw = (g * n).reshape(-1, n.shape[-1]).sum(0).to(weight.dtype)
        g = g * weight.float()
        dx = inv.unsqueeze(-1) * (g - n * (g * n).mean(-1, keepdim=True))
        dx = (dx if dsum is None else dx + dsum.float()).to(s.dtype)
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """y, or with a residual (y, s), s = x + residual rounded to x's type; both
    differentiable.  `weight` is of x's type or fp32."""
    if x.is_cuda:  # checked there, as below
        out = _backend.ext().rms_norm(x, weight, residual, eps)
        return out[0] if residual is None else tuple(out)
    _check(x, weight, residual)
    return _RMSNormFn.apply(x, weight, residual, float(eps))


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: Optional[torch.Tensor] = None, *,
                 eps: float = 1e-6, group: int = 0) -> Tuple[torch.Tensor, ...]:
    """The same norm with its output in e4m3: (codes, scales), or with a residual
    (codes, scales, s).  codes * scales is y: scales is fp32 [..., 1] with
    group = 0 (one scale a row) and [..., D / group] otherwise, each the largest
    magnitude it covers over 448.  `group` is a power of two from 16 to 512 that
    divides D.  A row that holds NaN gets NaN codes and scales.  No gradient:
    inputs that require one are refused while gradients are recorded."""
    if x.is_cuda:  # checked there, as below
        return tuple(_backend.ext().rms_norm_fp8(x, weight, residual, eps, group))
    _check(x, weight, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    D, lead = x.shape[-1], x.shape[:-1]
    if group != 0 and (group < 16 or group > 512 or group & (group - 1) or D % group):
        raise ValueError(f"rms_norm_fp8: group {group} is not a power of two from 16 to 512 that divides {D}")
    s = x if residual is None else x + residual
    sf = s.float().contiguous()
    y = sf * torch.rsqrt(sf.square().mean(-1, keepdim=True) + eps) * weight.float()
    y = y.view(*lead, D // (group or D), group or D)
    scales = (y.abs().amax(-1, keepdim=True) / _FP8_MAX).clamp_min(_TINY)
    codes = (y / scales).clamp(-_FP8_MAX, _FP8_MAX).to(_FP8).view(x.shape)
    out = (codes, scales.squeeze(-1))
    return out if residual is None else out + (s,)


class RMSNorm(nn.Module):
    """`rms_norm` with a learned weight, in a module's place for LayerNorm."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):  # noqa: D102
        return rms_norm(x, self.weight, residual, eps=self.eps)

    def extra_repr(self) -> str:
        return f"{self.weight.numel()}, eps={self.eps}"
