"""Softmax attention whose scores may be capped by a tanh and get a bias by
distance, under document, causal and prefix masks; forward, backward, and one or
a few queries against a long cache.

    s_ij = scale * q_i . k_j ;  softcap c: s = c tanh(s / c) ;  s -= slope_h |i + off - j|
    off  = key length - query length: the last query stands at the last key
    seen = (document_i == document_j >= 0) and (not causal or j <= i + off or j < prefix_b)
    o_i  = sum over seen j of softmax_j(s_ij) v_j ;  0 where a query sees nothing

GPU tensors run csrc/attention.hip, which never writes the scores to memory; CPU
tensors the same math in torch.  Scores, softmax statistics and sums are fp32;
weights and score gradients are rounded to the inputs' type before the second
products, as the matrix instructions take them.  What a masked key, value or
gradient row holds, NaN and infinities too, has no influence.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _backend

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_WIDTH = 128
MIN_SOFTCAP, MAX_SOFTCAP_16, MAX_SOFTCAP_32 = 2.0 ** -20, 2.0 ** 10, 2.0 ** 20


# ---------------------------------------------------------------------------
# torch (CPU) implementation
# ---------------------------------------------------------------------------

def _seen(Lq, Lk, B, causal, prefix, q_doc, k_doc, device):
    j = torch.arange(Lk, device=device)
    seen = torch.ones(B, Lq, Lk, dtype=torch.bool, device=device)
    if causal:
        end = (torch.arange(Lq, device=device) + (Lk - Lq + 1)).expand(B, Lq)
        if prefix is not None:
            end = torch.maximum(end, prefix.long()[:, None])
        seen = seen & (j < end[..., None])
    if q_doc is not None:
        seen = seen & (q_doc[:, :, None] == k_doc[:, None, :]) & (k_doc >= 0)[:, None, :]
    return seen[:, None]


def _masked_product(w, x, seen):
    """w @ x over what is seen (w is 0 elsewhere), whatever x holds elsewhere."""
    if torch.isfinite(x).all():
        return w @ x
    return torch.where(seen.unsqueeze(-1), w.unsqueeze(-1) * x.unsqueeze(-3), 0.0).sum(-2)


def _scores(q, k, scale, softcap, slopes, seen):
    s = (q @ k.transpose(-1, -2).contiguous()) * scale
    bend = None
    if softcap:
        t = torch.tanh(s / softcap)
        s, bend = softcap * t, 1 - t * t
    if slopes is not None:
        Lq, Lk = s.shape[-2:]
        at = torch.arange(Lq, device=s.device)[:, None] + (Lk - Lq)
        s = s - slopes.view(-1, 1, 1) * (at - torch.arange(Lk, device=s.device)).abs()
    return s.masked_fill(~seen, -math.inf), bend


def _heads(x, repeat=1):
    return x.float().transpose(1, 2).repeat_interleave(repeat, 1)


def _forward_torch(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc):
    G = q.shape[2] // k.shape[2]
    seen = _seen(q.shape[1], k.shape[1], q.shape[0], causal, prefix, q_doc, k_doc, q.device)
    s, _ = _scores(_heads(q), _heads(k, G), scale, softcap, slopes, seen)
    top = s.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = e.sum(-1, keepdim=True)
    none = ~seen.any(-1, keepdim=True)
    o = torch.where(none, 0.0, _masked_product(e, _heads(v, G), seen) / total)
    lse = torch.where(none, math.inf, top + total.log()).squeeze(-1)
    return o.transpose(1, 2).to(q.dtype).contiguous(), lse


def _backward_torch(g, q, k, v, o, lse, scale, softcap, slopes, causal, prefix, q_doc, k_doc):
    B, Lk, Hk, D = k.shape
    G = q.shape[2] // Hk
    seen = _seen(q.shape[1], Lk, B, causal, prefix, q_doc, k_doc, q.device)
    qf, kf, vf, gf = _heads(q), _heads(k, G), _heads(v, G), _heads(g)
    s, bend = _scores(qf, kf, scale, softcap, slopes, seen)
    p = torch.where(seen, torch.exp(s - lse.unsqueeze(-1)), 0.0)
    delta = (gf * _heads(o)).sum(-1, keepdim=True)
    ds = p * (gf @ vf.transpose(-1, -2).contiguous() - delta) * scale
    ds = torch.where(seen, ds if bend is None else ds * bend, 0.0)
    back = seen.transpose(-1, -2)
    turned = lambda x: x.transpose(-1, -2).contiguous()  # noqa: E731
    dq = _masked_product(ds, kf, seen)
    dk, dv = _masked_product(turned(ds), qf, back), _masked_product(turned(p), gf, back)
    dk, dv = (x.view(B, Hk, G, Lk, D).sum(2) for x in (dk, dv))
    return [x.transpose(1, 2).to(q.dtype).contiguous() for x in (dq, dk, dv)]


# ---------------------------------------------------------------------------
# autograd binding
# ---------------------------------------------------------------------------

class _AttentionFn(torch.autograd.Function):
    """On the CPU, and where there is nothing to attend to; GPU tensors are recorded in
    csrc/autograd.cpp."""

    @staticmethod
    def forward(ctx, q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc):
        ctx.how = (scale, softcap, causal)
        ctx.empty = q.numel() == 0 or k.numel() == 0
        if ctx.empty:
            ctx.save_for_backward(q, k, v)
            return torch.zeros_like(q, memory_format=torch.contiguous_format)
        o, lse = _forward_torch(q, k, v, scale, softcap, slopes, causal, prefix, q_doc, k_doc)
        ctx.save_for_backward(q, k, v, o, lse, slopes, prefix, q_doc, k_doc)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        if ctx.empty:
            return tuple(torch.zeros_like(x) for x in ctx.saved_tensors) + (None,) * 7
        q, k, v, o, lse, slopes, prefix, q_doc, k_doc = ctx.saved_tensors
        scale, softcap, causal = ctx.how
        return tuple(_backward_torch(g, q, k, v, o, lse, scale, softcap, slopes, causal, prefix, q_doc, k_doc)) + (None,) * 7


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, scale: Optional[float] = None, softcap: float = 0.0,
              slopes: Optional[torch.Tensor] = None, causal: bool = False, prefix: Optional[torch.Tensor] = None,
              documents: Optional[torch.Tensor] = None, key_documents: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[batch, queries, heads, width] from q of that shape and k, v [batch, keys,
    key heads, width]; key heads divide heads, and head h reads key head
    h // (heads / key heads).  fp32, bf16 or fp16, widths up to 128, any strides;
    differentiable in q, k and v.

    `scale` is width^-0.5 by default.  `softcap` 0 leaves scores as they are; others
    lie from 2^-20 to 2^20 (16-bit types: 2^10, as the cap is formed to 8 units of it).
    `slopes` fp32 [heads] biases by distance (no gradient).  `causal` hides keys
    behind the query's place, but for the first `prefix[b]` (int32 [batch]) keys.
    `documents` int32 [batch, queries] and `key_documents` [batch, keys] (the same
    where it is left out and the lengths agree) let a query see keys of its own
    id, in any order; negative ids are padding: such queries see nothing, such
    keys are seen by none.  GPU calls take under 2^24 tiles of 128 queries or keys,
    over batch and heads."""
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.dim() != 4:
            raise ValueError(f"attention: {name} is [batch, length, heads, width], got {tuple(x.shape)}")
        if x.dtype not in _FLOATS or x.dtype != q.dtype:
            raise TypeError(f"attention: q, k and v are fp32, bf16 or fp16 of one type, got {name} {x.dtype}")
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    if v.shape != k.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not go together")
    if not 1 <= D <= MAX_WIDTH:
        raise ValueError(f"attention: widths of 1 to {MAX_WIDTH} expected, got {D}")
    if Hk == 0 or H % Hk:
        raise ValueError(f"attention: {Hk} key heads do not divide {H} heads")
    scale = D ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 2.0 ** 100:
        raise ValueError(f"attention: a scale of at most 2^100 expected, got {scale}")
    most = MAX_SOFTCAP_32 if q.dtype == torch.float32 else MAX_SOFTCAP_16
    if not (softcap == 0.0 or MIN_SOFTCAP <= softcap <= most):
        raise ValueError(f"attention: a softcap of 0 or {MIN_SOFTCAP:g} to {most:g} expected for {q.dtype}, got {softcap}")
    if slopes is not None:
        if slopes.shape != (H,) or slopes.dtype != torch.float32:
            raise ValueError(f"attention: slopes are fp32 [{H}], got {slopes.dtype} {tuple(slopes.shape)}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("attention: slopes have no gradient")
    if prefix is not None and not causal:
        raise ValueError("attention: a prefix goes with causal=True")
    if key_documents is None and documents is not None:
        if Lq != Lk:
            raise ValueError(f"attention: {Lq} queries and {Lk} keys need key_documents")
        key_documents = documents
    if key_documents is not None and documents is None:
        raise ValueError("attention: key_documents go with documents")
    for name, x, shape in (("prefix", prefix, (B,)), ("documents", documents, (B, Lq)), ("key_documents", key_documents, (B, Lk))):
        if x is not None and (tuple(x.shape) != shape or x.dtype != torch.int32):
            raise ValueError(f"attention: {name} is int32 {list(shape)}, got {x.dtype} {tuple(x.shape)}")
    for x in (k, v, slopes, prefix, documents, key_documents):
        if x is not None and x.device != q.device:
            raise ValueError(f"attention: tensors on {q.device} and {x.device}")
    slopes, prefix, documents, key_documents = (x if x is None else x.detach().contiguous()
                                                for x in (slopes, prefix, documents, key_documents))
    args = (q, k, v, scale, float(softcap), slopes, bool(causal), prefix, documents, key_documents)
    if q.is_cuda and q.numel() and k.numel():
        return _backend.ext().attention(*args)
    return _AttentionFn.apply(*args)
