"""Rotary positions: pair i of a head's leading elements is turned by the angle
position * frequency_i, so that products of queries and keys go by the distance
between their positions.

Two layouts of the pairs (element i with element i + pairs, or interleaved
neighbours), any leading part of the head, positions along one axis or several
(rows and columns of an image's patches), frequencies scaled for long contexts.
GPU tensors run csrc/rotary.hip, one launch for q and k; CPU tensors the same
math in torch.  Angles are formed in fp64 whatever the inputs' type.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from . import _backend

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_PAIRS = 512
MAX_HEADS = MAX_WIDTH = 4096  # heads of q and k together
SCALINGS = (None, "linear", "base", "ramp")


def rotary_frequencies(dim: int, *, axes: int = 1, base: float = 10000.0, scaling: Optional[str] = None,
                       factor: float = 1.0, original_length: int = 0, fast_turns: float = 32.0,
                       slow_turns: float = 1.0, device=None) -> Tuple[torch.Tensor, float]:
    """(frequencies, amplitude) for `dim` elements of a head over `axes` position
    axes.  frequencies is fp64: [dim / 2], or [axes, dim / (2 axes)] for axes > 1,
    base^(-i / n) for i of the n pairs of an axis.

    `scaling` stretches them for contexts `factor` times as long:
      "linear"  every frequency over factor (positions are squeezed);
      "base"    the base grows so that the slowest pair slows by factor and the
                fastest stays;
      "ramp"    pairs that turn more than `fast_turns` times within
                `original_length` stay, ones under `slow_turns` slow by factor,
                a linear ramp between; amplitude becomes 0.1 ln(factor) + 1.
    amplitude is 1 otherwise."""
    if axes < 1 or dim < 2 * axes or dim % (2 * axes):
        raise ValueError(f"rotary_frequencies: dim {dim} is not a multiple of 2 * {axes} axes")
    if scaling not in SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling {scaling!r} is none of {SCALINGS}")
    if not factor >= 1.0 or not base > 1.0:
        raise ValueError(f"rotary_frequencies: factor >= 1 and base > 1 expected, got {factor}, {base}")
    n = dim // (2 * axes)
    amplitude = 1.0
    if scaling == "base" and n > 1:
        base = base * factor ** (n / (n - 1))
    f = base ** (-torch.arange(n, dtype=torch.float64) / n)
    if scaling == "linear":
        f = f / factor
    elif scaling == "ramp":
        if original_length < 1 or not fast_turns > slow_turns > 0:
            raise ValueError("rotary_frequencies: ramp needs original_length and fast_turns > slow_turns > 0")
        turns = original_length * f / (2 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    f = f if axes == 1 else f.expand(axes, n).contiguous()
    return f.to(device), amplitude


def _turn_torch(x, angle, interleaved, amplitude, backward):
    c, z = ((fn(angle) * amplitude).float().unsqueeze(2) for fn in (torch.cos, torch.sin))
    z = -z if backward else z
    P, xf = angle.shape[-1], x.float()
    head, rest = xf[..., :2 * P], xf[..., 2 * P:]
    a, b = (head[..., 0::2], head[..., 1::2]) if interleaved else (head[..., :P], head[..., P:])
    u, v = a * c - b * z, a * z + b * c
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, rest], -1).to(x.dtype)


def _turn(q, k, positions, frequencies, interleaved, amplitude, backward):
    f = frequencies.reshape(positions.shape[-1], -1)
    angle = (positions.double().unsqueeze(-1) * f).flatten(-2)
    return [_turn_torch(x, angle, interleaved, amplitude, backward) for x in (q, k) if x is not None]


class _RotaryFn(torch.autograd.Function):
    """On the CPU; GPU tensors are recorded in csrc/autograd.cpp."""

    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, amplitude):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (interleaved, amplitude)
        ctx.set_materialize_grads(False)
        out = _turn(q, k, positions, frequencies, interleaved, amplitude, False)
        return out[0] if k is None else tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk=None):
        grads = [g for g in (dq, dk) if g is not None]
        if not grads:
            return (None,) * 6
        got = iter(_turn(grads[0], grads[1] if len(grads) > 1 else None, *ctx.saved_tensors, *ctx.how, True))
        return (None if dq is None else next(got), None if dk is None else next(got), None, None, None, None)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, *,
           interleaved: bool = False, amplitude: float = 1.0) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """q [batch, length, heads, width], and k with heads of its own (or None), with
    the first 2 * frequencies.numel() elements of every head turned; contiguous,
    differentiable in q and k.  Up to 4096 heads of both together, widths up to 4096,
    512 frequencies (on the GPU under 2^24 blocks of up to 16 tokens).  `positions` is int32 or int64: [length] or
    [batch, length], with one more dimension of axes where `frequencies` is
    [axes, n] (axis a turns pairs a n to a n + n).  `frequencies` is fp64, from
    `rotary_frequencies`, and gets no gradient; cosines and sines are multiplied by
    `amplitude`."""
    if q.is_cuda:  # checked there, as below
        out = _backend.ext().rotary(q, k, positions, frequencies, interleaved, amplitude)
        return out[0] if k is None else tuple(out)
    for name, x in (("q", q), ("k", k)):
        if x is None:
            continue
        if x.dim() != 4:
            raise ValueError(f"rotary: {name} is [batch, length, heads, width], got {tuple(x.shape)}")
        if x.dtype not in _FLOATS or x.dtype != q.dtype:
            raise TypeError(f"rotary: q and k are fp32, bf16 or fp16 of one type, got {name} {x.dtype}")
        if x.shape[:2] != q.shape[:2] or x.shape[3] != q.shape[3]:
            raise ValueError(f"rotary: q {tuple(q.shape)} and k {tuple(x.shape)} do not go together")
    heads = q.shape[2] + (0 if k is None else k.shape[2])
    if heads > MAX_HEADS or q.shape[3] > MAX_WIDTH:
        raise ValueError(f"rotary: up to {MAX_HEADS} heads of q and k together and widths up to {MAX_WIDTH} expected, got {heads} of {q.shape[3]}")
    if frequencies.dtype != torch.float64 or frequencies.dim() not in (1, 2):
        raise TypeError(f"rotary: frequencies are fp64 [n] or [axes, n], got {frequencies.dtype} {tuple(frequencies.shape)}")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("rotary: frequencies have no gradient")
    P = frequencies.numel()
    if not 1 <= P <= MAX_PAIRS or 2 * P > q.shape[3]:
        raise ValueError(f"rotary: {P} frequencies do not fit heads of {q.shape[3]} (at most {MAX_PAIRS})")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"rotary: positions are int32 or int64, got {positions.dtype}")
    lead = positions.shape[:-1] if frequencies.dim() == 2 else positions.shape
    axes = positions.shape[-1:] if frequencies.dim() == 2 else (1,)
    if tuple(lead) not in (tuple(q.shape[1:2]), tuple(q.shape[:2])) or (frequencies.dim() == 2 and axes[0] != frequencies.shape[0]):
        raise ValueError(f"rotary: positions {tuple(positions.shape)} do not fit q {tuple(q.shape)} and "
                         f"frequencies {tuple(frequencies.shape)}")
    for t in (k, positions, frequencies):
        if t is not None and t.device != q.device:
            raise ValueError(f"rotary: tensors on {q.device} and {t.device}")
    positions = positions.reshape(*lead, *axes).expand(q.shape[0], q.shape[1], *axes)
    return _RotaryFn.apply(q, k, positions, frequencies, bool(interleaved), float(amplitude))
