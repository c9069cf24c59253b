"""One AdamW step over many tensors, with moments in fp32 or in 8 bits.

    m = b1 m + (1 - b1) g            v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

In 8 bits blocks of 256 elements share an fp32 scale; m and the root of v are
e4m3 codes, rounded stochastically (unbiased in m and in v) by bits that are a
hash of seed, step, tensor, block and element, so that equal calls give equal
codes.  GPU tensors run csrc/adamw.hip; CPU tensors the same steps in torch,
with the same codes.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import _backend

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_FP8 = torch.float8_e4m3fn
_FP8_MAX = 448.0
_MIN_NORMAL = 2.0 ** -6
_TINY = 2.0 ** -126
BLOCK = 256


def _like(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors of one shape lie in memory in the same order."""
    return all(n <= 1 or s == t for n, s, t in zip(b.shape, a.stride(), b.stride()))


def _dense(p: torch.Tensor) -> bool:
    """Whether a tensor's elements fill one stretch of memory, in any order of dimensions."""
    expect = 1
    for s, n in sorted((s, n) for s, n in zip(p.stride(), p.shape) if n != 1):
        if s != expect:
            return p.numel() == 0
        expect *= n
    return True


def adamw_state(param: torch.Tensor, *, bits: int = 32, master: bool = False) -> dict:
    """Fresh state for one parameter: exp_avg, exp_avg_sq (with bits=8 e4m3 codes,
    of the root in the second, and their `scales` [blocks, 2]), `step` (int32 on
    the device) and, where asked for and the parameter is not fp32, `master`."""
    if bits not in (8, 32):
        raise ValueError(f"adamw: moments in 8 or 32 bits, got {bits}")
    if param.dtype not in _FLOATS:
        raise TypeError(f"adamw: fp32, bf16 or fp16 parameters expected, got {param.dtype}")
    if not _dense(param):
        raise ValueError(f"adamw: a parameter fills a stretch of memory, got strides {param.stride()} for {tuple(param.shape)}")
    zeros = torch.zeros_like(param, dtype=torch.uint8).view(_FP8) if bits == 8 else torch.zeros_like(param, dtype=torch.float32)
    state = {"step": torch.zeros((), dtype=torch.int32, device=param.device), "exp_avg": zeros, "exp_avg_sq": zeros.clone()}
    if bits == 8:
        state["scales"] = torch.zeros((param.numel() + BLOCK - 1) // BLOCK, 2, device=param.device)
    if master and param.dtype != torch.float32:
        state["master"] = param.detach().float()
    return state


def _check(params, grads, exp_avgs, exp_avg_sqs, steps, masters, scales) -> List[torch.Tensor]:
    """The gradients, in the order of their parameters in memory."""
    device, dtype = params[0].device, params[0].dtype
    if dtype not in _FLOATS:
        raise TypeError(f"adamw_step: fp32, bf16 or fp16 parameters expected, got {dtype}")
    state = _FP8 if scales is not None else torch.float32
    laid: List[torch.Tensor] = []
    for i, (p, g, m, v, t) in enumerate(zip(params, grads, exp_avgs, exp_avg_sqs, steps)):
        if p.device != device or p.dtype != dtype:
            raise ValueError(f"adamw_step: parameter {i} is {p.dtype} on {p.device}, the first {dtype} on {device}")
        if not _dense(p):
            raise ValueError(f"adamw_step: parameter {i} does not fill a stretch of memory (strides {p.stride()})")
        if g.layout != torch.strided or g.shape != p.shape or g.dtype != dtype or g.device != device:
            raise ValueError(f"adamw_step: gradient {i} {tuple(g.shape)} {g.dtype} does not fit {tuple(p.shape)} {dtype}")
        for name, x, want in (("exp_avg", m, state), ("exp_avg_sq", v, state)) + ((("master", masters[i], torch.float32),) if masters is not None else ()):
            if x.shape != p.shape or x.dtype != want or x.device != device or not _like(x, p):
                raise ValueError(f"adamw_step: {name} {i} {tuple(x.shape)} {x.dtype} is not laid out as its parameter in {want}")
        if t.numel() != 1 or t.dtype != torch.int32 or t.device != device:
            raise ValueError(f"adamw_step: step {i} is one int32 on {device}")
        if scales is not None and (scales[i].shape != ((p.numel() + BLOCK - 1) // BLOCK, 2) or scales[i].dtype != torch.float32
                                   or scales[i].device != device or not scales[i].is_contiguous()):
            raise ValueError(f"adamw_step: scales {i} {tuple(scales[i].shape)} are not fp32 [blocks of {BLOCK}, 2]")
        laid.append(g if _like(g, p) else torch.empty_like(p).copy_(g))
    written = sorted((x.data_ptr(), x.data_ptr() + x.numel() * x.element_size())
                     for xs in (params, exp_avgs, exp_avg_sqs, steps, masters or (), scales or ()) for x in xs if x.numel())
    if any(a[1] > b[0] for a, b in zip(written, written[1:])):
        raise RuntimeError("adamw_step: a tensor comes twice, or overlaps another")
    return laid


def adamw_step(params: Sequence[torch.Tensor], grads: Sequence[torch.Tensor], exp_avgs: Sequence[torch.Tensor],
               exp_avg_sqs: Sequence[torch.Tensor], steps: Sequence[torch.Tensor], *, lr: float,
               betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               masters: Optional[Sequence[torch.Tensor]] = None, scales: Optional[Sequence[torch.Tensor]] = None,
               seed: int = 0) -> None:
    """Updates every list in place; state as `adamw_state` makes it.

    The parameters are of one type on one device and dense in memory, a gradient
    of its parameter's type; one that lies in another order is copied first.  What is
    updated comes once: tensors that share memory are refused, steps too.
    `steps` counts the steps done, one int32 on the device a tensor, read and
    raised there (a captured step counts on).  With `masters` (fp32) they are
    updated and the parameters rounded from them; with `scales` the moments are
    in 8 bits and `seed` chooses the random bits.  `lr`, `betas`, `eps` and
    `weight_decay` are the host's: a captured step keeps them."""
    lists = [params, grads, exp_avgs, exp_avg_sqs, steps] + [x for x in (masters, scales) if x is not None]
    if len({len(x) for x in lists}) != 1:
        raise ValueError(f"adamw_step: lists of different lengths: {[len(x) for x in lists]}")
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
        raise ValueError(f"adamw_step: betas in [0, 1) expected, got {betas}")
    if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0):
        raise ValueError(f"adamw_step: lr, eps and weight_decay are not negative, got {lr}, {eps}, {weight_decay}")
    if not len(params):
        return
    with torch.no_grad():
        if params[0].device.type == "cuda":  # checked there, as below
            _backend.ext().adamw_update(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), list(steps), list(masters or ()),
                                        list(scales or ()), float(lr), float(betas[0]), float(betas[1]), float(eps),
                                        float(weight_decay), int(seed) & 0xFFFFFFFF)
            return
        laid = _check(params, grads, exp_avgs, exp_avg_sqs, steps, masters, scales)
        for i, (p, g, m, v, t) in enumerate(zip(params, laid, exp_avgs, exp_avg_sqs, steps)):
            _step_torch(p, g, m, v, t, masters[i] if masters is not None else None, scales[i] if scales is not None else None,
                        lr, betas, eps, weight_decay, int(seed) & 0xFFFFFFFF, i)


# ---------------------------------------------------------------------------
# torch (CPU) implementation: the operations of csrc/adamw.hip, one by one
# ---------------------------------------------------------------------------

def _mix(x: torch.Tensor) -> torch.Tensor:
    x = ((x ^ (x >> 16)) * 0x9E3779B9) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xB7E15163) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _bits(seed: int, step: int, tensor: int, blocks: int) -> torch.Tensor:
    key = _mix(torch.tensor((seed + step * 0x9E3779B9) & 0xFFFFFFFF)) ^ ((tensor * 0xB7E15163) & 0xFFFFFFFF)
    key = _mix(_mix(key) ^ torch.arange(blocks))
    return _mix((key[:, None] + torch.arange(BLOCK) * 0x9E3779B9) & 0xFFFFFFFF)


def _memory_order(x: torch.Tensor) -> torch.Tensor:
    """A dense tensor's elements in the order of their addresses, as a view."""
    return x.as_strided((x.numel(),), (1,))


def _blocks(x: torch.Tensor) -> torch.Tensor:
    x = _memory_order(x).float()
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _offset(a):
    return torch.where(a < _MIN_NORMAL, _MIN_NORMAL, 0.0)


def _step_torch(p, g, m, v, t, master, scale, lr, betas, eps, weight_decay, seed, index):
    b1, b2 = betas
    t.add_(1)
    step = int(t)
    w = p if master is None else master
    if scale is None:
        gf = g.float()
        m.mul_(b1).add_(gf, alpha=1 - b1)
        v.mul_(b2).addcmul_(gf, gf, value=1 - b2)
        new_m, root = m, v.sqrt()
    else:
        gb, mb, rb = _blocks(g), _blocks(m) * scale[:, :1], _blocks(v) * scale[:, 1:]
        mb = mb * b1 + gb * (1 - b1)
        # a correctly rounded fp32 root, as the GPU's: torch's own on the CPU is off by a unit on some machines
        rb = torch.sqrt(((rb * rb) * b2 + (gb * gb) * (1 - b2)).double()).float()
        for i, x in enumerate((mb, rb)):
            top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(1)
            scale[:, i] = (top * (1.0 / _FP8_MAX)).clamp_min(_TINY)
        inverse = 1.0 / scale
        bits = _bits(seed, step, index, mb.shape[0])
        x = mb * inverse[:, :1]
        a = x.abs().clamp_max(_FP8_MAX)
        low = _offset(a)
        up = (((a + low).view(torch.int32) + (((bits & 0xFFFF) << 4) | 8).int()) & ~0xFFFFF).view(torch.float32) - low
        code_m = torch.where(torch.isfinite(mb), torch.copysign(up.clamp_max(_FP8_MAX), x), float("nan"))
        a = (rb * inverse[:, 1:]).clamp_max(_FP8_MAX)
        low = _offset(a)
        cut = (a + low).view(torch.int32) & ~0xFFFFF
        down, up = cut.view(torch.float32) - low, (cut + 0x100000).view(torch.float32) - low
        chance = ((bits >> 16).float() + 0.5) * 2.0 ** -16
        r = torch.where(chance * ((up - down) * (up + down)) < (a - down) * (a + down), up, down).clamp_max(_FP8_MAX)
        r = torch.where((a > 0) & (r == 0), 2.0 ** -9, r)
        code_v = torch.where(torch.isfinite(rb), r, float("nan"))
        n = p.numel()
        for state, code in ((m, code_m), (v, code_v)):
            _memory_order(state).copy_(code.view(-1)[:n].to(_FP8))
        new_m, root = (torch.empty_like(w, dtype=torch.float32).as_strided((n,), (1,)).copy_(x.view(-1)[:n]).as_strided(w.shape, w.stride())
                       for x in (mb, rb))
    c1, c2 = 1 - b1 ** step, 1 - b2 ** step
    new = w.float() * (1 - lr * weight_decay) - (lr / c1) * (new_m / (root / c2 ** 0.5 + eps))
    w.copy_(new)
    if master is not None:
        p.copy_(master)
