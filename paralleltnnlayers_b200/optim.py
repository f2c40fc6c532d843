"""Optimiser over the fused AdamW step: what applies the gradients of the layers and of the data-parallel steps.

A network of factored layers has many small parameters (four factors per convolution); all of them are updated by one launch.
"""
from __future__ import annotations

from itertools import chain

import torch

BLOCK = 256   # values of 8-bit moments that share a scale


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with ``torch.optim.AdamW``'s arguments, its update in fp32.

    ``bits=8`` keeps the moments as 8-bit codes with a float32 scale per 256 values: 2.03 bytes a value instead of 8.  16-bit
    parameters get a float32 copy that is what is updated (``master=False``: the parameter itself, rounded at each step).
    ``capturable=True`` keeps a count of the steps on the device, one for all parameters of a group, so that a captured ``step()``
    counts its replays; make one step before the capture.  ``lr`` may be one float32 in a CUDA tensor.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32, master=True, capturable=False):
        if bits not in (8, 32):
            raise ValueError("moments are held in 8 or 32 bits")
        if not torch.is_tensor(lr) and lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr, eps and weight_decay may not be negative, betas are in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits, master=master, capturable=capturable))

        self._counts = {}

    def _state_of(self, p, at, group):
        s = self.state[p]
        if not s:
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise TypeError(f"parameters are float32, bfloat16 or float16, not {p.dtype}")
            if not p.is_contiguous():
                raise ValueError("parameters are updated in place and have to be contiguous")
            s["step"] = self._count(at, p.device) if group["capturable"] else 0
            if group["bits"] == 8:
                blocks = (p.numel() + BLOCK - 1) // BLOCK
                s["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8, device=p.device)
                s["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
                s["scale_avg"], s["scale_sq"] = (torch.zeros(blocks, dtype=torch.float32, device=p.device) for _ in range(2))
            else:
                s["exp_avg"], s["exp_avg_sq"] = (torch.zeros(p.shape, dtype=torch.float32, device=p.device) for _ in range(2))
            if group["master"] and p.dtype != torch.float32:
                s["master"] = p.detach().float()
        return s

    def _count(self, at, device):
        """The steps of a group's parameters on a device, on that device."""
        if (at, device) not in self._counts:
            self._counts[at, device] = torch.zeros((), dtype=torch.int64, device=device)
        return self._counts[at, device]

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every parameter that has a gradient, a launch per type and device (and per count of steps, where some
        parameters had no gradient in earlier steps)."""
        from . import ops
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for at, group in enumerate(self.param_groups):
            calls, counted = {}, set()
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise TypeError("gradients have to be dense")
                s = self._state_of(p, at, group)
                if group["capturable"]:
                    counted.add(p.device)
                    count = None
                else:
                    s["step"] += 1
                    count = s["step"]
                calls.setdefault((p.device, p.dtype, p.grad.dtype, "master" in s, count), []).append((p, s))
            for device in counted:
                self._count(at, device).add_(1)
            for (device, _, _, copies, count), members in calls.items():
                ps, ss = zip(*members)
                ops.adamw_step([p.detach() for p in ps], [p.grad for p in ps], [s["exp_avg"] for s in ss], [s["exp_avg_sq"] for s in ss],
                               self._count(at, device) if count is None else count, group["lr"], group["betas"], group["eps"],
                               group["weight_decay"], [s["master"] for s in ss] if copies else None,
                               ([s["scale_avg"] for s in ss], [s["scale_sq"] for s in ss]) if group["bits"] == 8 else None)
        return loss

    def __setstate__(self, state):
        """A copied or unpickled optimiser: the parameters of a group share its count again."""
        super().__setstate__(state)
        self._counts = {}
        for at, group in enumerate(self.param_groups):
            for p in group["params"]:
                s = self.state.get(p)
                if group["capturable"] and s and torch.is_tensor(s.get("step")):
                    s["step"] = self._counts.setdefault((at, p.device), s["step"])

    def load_state_dict(self, state_dict):
        """As the base class, but the state keeps its own types (codes, float32 moments of 16-bit parameters)."""
        super().load_state_dict(state_dict)
        names = chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        self._counts = {}
        of = {id(p): at for at, g in enumerate(self.param_groups) for p in g["params"]}
        for name, p in zip(names, chain.from_iterable(g["params"] for g in self.param_groups)):
            if name not in state_dict["state"]:
                continue
            s = {k: v.detach().to(p.device, copy=True) if torch.is_tensor(v) else v for k, v in state_dict["state"][name].items()}
            at = of[id(p)]
            if self.param_groups[at]["capturable"]:
                count = self._count(at, p.device)
                count.copy_(torch.as_tensor(s["step"]))
                s["step"] = count
            elif torch.is_tensor(s["step"]):
                s["step"] = int(s["step"])
            self.state[p] = s
