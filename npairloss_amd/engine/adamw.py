"""AdamW as a solver beside CaffeSGD, on `ops.adamw_step` (csrc/adamw.hip).

One step is a few launches for all tensors of a group, however many there are.
Counts of steps live on the device, so a hipGraph that holds a step counts on
when it is replayed; lr is the host's, as CaffeSGD's is, and a captured step
keeps it.  `state_bits=8` holds both moments in 8 bits (2 bytes a parameter in
place of 8, and 8 for every 256), `master_weights=True` keeps fp32 masters of
16-bit parameters.
"""

from __future__ import annotations

from typing import Iterable, Tuple

import torch

from ..ops.adamw import adamw_state, adamw_step


class AdamW(torch.optim.Optimizer):
    """Parameters whose gradient is None are left alone and their step is not
    counted.  `seed` chooses the random bits that 8-bit moments are rounded by;
    a run is repeated by the same seed."""

    def __init__(self, params: Iterable, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, master_weights: bool = False,
                 state_bits: int = 32, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: moments in 8 or 32 bits, got {state_bits}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"AdamW: betas in [0, 1) expected, got {betas}")
        if not (lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0):
            raise ValueError(f"AdamW: lr, eps and weight_decay are not negative, got {lr}, {eps}, {weight_decay}")
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay,
                                      master_weights=master_weights, state_bits=state_bits, seed=seed))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for number, group in enumerate(self.param_groups):
            lists = {}  # by device and type: one call takes tensors of one kind
            for place, p in enumerate(group["params"]):
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("AdamW: sparse gradients are not supported")
                st = self.state[p]
                if not st:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: make one step before capturing one: the state would be made anew at every replay")
                    st.update(adamw_state(p, bits=group["state_bits"], master=group["master_weights"]))
                lists.setdefault((p.device, p.dtype), []).append((place, p, st))
            for kind, ((_, dtype), found) in enumerate(lists.items()):
                places, ps, sts = zip(*found)
                masters = [st["master"] for st in sts] if "master" in sts[0] else None
                scales = [st["scales"] for st in sts] if group["state_bits"] == 8 else None
                adamw_step(ps, [p.grad for p in ps], [st["exp_avg"] for st in sts], [st["exp_avg_sq"] for st in sts],
                           [st["step"] for st in sts], lr=group["lr"], betas=group["betas"], eps=group["eps"],
                           weight_decay=group["weight_decay"], masters=masters, scales=scales,
                           seed=group["seed"] + 0x3779 * number + 0x51 * kind)
        return loss

    def set_lr(self, lr: float):
        for group in self.param_groups:
            group["lr"] = lr

    def load_state_dict(self, state_dict):
        """Optimizer.load_state_dict turns floating state into the parameter's type;
        this one's keeps its own (codes, fp32 moments, masters, counts)."""
        super().load_state_dict(state_dict)
        saved = state_dict["state"]
        index = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(index, params):
            if i in saved:
                self.state[p] = {k: v.detach().clone().to(p.device) if torch.is_tensor(v) else v for k, v in saved[i].items()}
