"""Optimisers over the fused AdamW and Muon steps: what applies the gradients of the layers and of the data-parallel steps.

A network of factored layers has many small parameters (four factors per convolution); all of them are updated by one launch (three for
Muon, and 18 more where a matrix has both sides above 64).
"""
from __future__ import annotations

from itertools import chain

import torch

BLOCK = 256   # values of 8-bit moments that share a scale


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) with ``torch.optim.AdamW``'s arguments, its update in fp32.

    ``bits=8`` keeps the moments as 8-bit codes with a float32 scale per 256 values: 2.03 bytes a value instead of 8.  16-bit
    parameters get a float32 copy that is what is updated (``master=False``: the parameter itself, rounded at each step); it is taken at a
    parameter's first step, so values that are put into the parameter later do not reach it.
    ``capturable=True`` keeps the counts of steps on the device, one for all parameters that have taken the same steps, so that a captured
    ``step()`` counts its replays; make one step with the same gradients before the capture.  (A step that would begin a state or a count
    inside a capture is refused: each replay would begin it again.)  ``lr`` may be one float32 in a CUDA tensor.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, bits=32, master=True, capturable=False):
        if bits not in (8, 32):
            raise ValueError("moments are held in 8 or 32 bits")
        if not torch.is_tensor(lr) and lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("lr, eps and weight_decay may not be negative, betas are in [0, 1)")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits, master=master, capturable=capturable))

    def _state_of(self, p, group, first, capturing):
        s = self.state[p]
        if not s:
            if capturing:
                raise RuntimeError("a captured step() begins no state: make a step with the same gradients before the capture")
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise TypeError(f"parameters are float32, bfloat16 or float16, not {p.dtype}")
            if not p.is_contiguous():
                raise ValueError("parameters are updated in place and have to be contiguous")
            if not group["capturable"]:
                s["step"] = 0
            else:   # parameters whose first step is the same share a count
                if p.device not in first:
                    first[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
                s["step"] = first[p.device]
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

    def _advance(self, group, members, capturing):
        """One step more for the counts of these states of a capturable group.  Parameters that share a count with others that have no gradient
        this time get one of their own."""
        counts, sharers = {}, {}
        for s in members:
            counts.setdefault(id(s["step"]), []).append(s)
        if len(members) < len(group["params"]):   # (else all that share a count are here)
            for p in group["params"]:
                s = self.state.get(p)
                if s:
                    sharers[id(s["step"])] = sharers.get(id(s["step"]), 0) + 1
        for at, ss in counts.items():
            count = ss[0]["step"]
            if len(ss) < sharers.get(at, 0):
                if capturing:
                    raise RuntimeError("a captured step() divides no count: make a step with the same gradients before the capture")
                count = count.clone()
                for s in ss:
                    s["step"] = count
            count.add_(1)

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every parameter that has a gradient, a launch per type and device (and per count of steps, where some
        parameters had no gradient in earlier steps)."""
        from . import ops
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        for group in self.param_groups:
            if capturing and not group["capturable"] and any(p.grad is not None for p in group["params"]):
                raise RuntimeError("a captured step() counts its replays with capturable=True alone")
            calls, stepped, first = {}, [], {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise TypeError("gradients have to be dense")
                s = self._state_of(p, group, first, capturing)
                if group["capturable"]:
                    stepped.append((p, s))
                else:
                    s["step"] += 1
                    calls.setdefault((p.device, p.dtype, p.grad.dtype, "master" in s, s["step"]), []).append((p, s))
            if stepped:
                self._advance(group, [s for _, s in stepped], capturing)
            for p, s in stepped:
                calls.setdefault((p.device, p.dtype, p.grad.dtype, "master" in s, id(s["step"])), []).append((p, s))
            for (_, _, _, copies, _), members in calls.items():
                ps, ss = zip(*members)
                ops.adamw_step([p.detach() for p in ps], [p.grad for p in ps], [s["exp_avg"] for s in ss], [s["exp_avg_sq"] for s in ss],
                               ss[0]["step"], group["lr"], group["betas"], group["eps"],
                               group["weight_decay"], [s["master"] for s in ss] if copies else None,
                               ([s["scale_avg"] for s in ss], [s["scale_sq"] for s in ss]) if group["bits"] == 8 else None)
        return loss

    def _share_counts(self):
        """Parameters of a capturable group that have taken as many steps share a count (where they took different ones, it divides later)."""
        for group in self.param_groups:
            counts = {}
            for p in group["params"]:
                s = self.state.get(p)
                if group["capturable"] and s and torch.is_tensor(s.get("step")):
                    s["step"] = counts.setdefault((p.device, int(s["step"])), s["step"])

    def __setstate__(self, state):
        """A copied or unpickled optimiser: parameters share their counts again."""
        super().__setstate__(state)
        self._share_counts()

    def load_state_dict(self, state_dict):
        """As the base class, but the state keeps its own types (codes, float32 moments of 16-bit parameters)."""
        super().load_state_dict(state_dict)
        names = chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        for name, (group, p) in zip(names, ((g, p) for g in self.param_groups for p in g["params"])):
            if name not in state_dict["state"]:
                continue
            s = {k: v.detach().to(p.device, copy=True) if torch.is_tensor(v) else v for k, v in state_dict["state"][name].items()}
            steps = int(s["step"])
            s["step"] = torch.full((), steps, dtype=torch.int64, device=p.device) if group["capturable"] else steps
            self.state[p] = s
        self._share_counts()


class Muon(torch.optim.Optimizer):
    """Muon for matrices: the momentum of each is orthogonalised by Newton-Schulz products before it is subtracted, with ``torch.optim.Muon``'s arguments.

    Parameters have two dimensions or more; leading ones are stacks of matrices (``AdaptedDense.A`` and ``.B``), each orthogonalised by itself.  Vectors (biases,
    norms) and embeddings belong to an ``AdamW`` beside it.  Momentum is float32.  16-bit parameters get a float32 copy that is what is updated
    (``master=False``: the parameter itself, rounded at each step); it is taken at a parameter's first step.  ``lr`` may be one float32 in a CUDA tensor.
    A captured ``step()`` begins no state: make one step with the same gradients before the capture.  A ``torch.optim.Muon``'s state can be loaded."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_coefficients=(3.4445, -4.7750, 2.0315), eps=1e-7, ns_steps=5,
                 adjust_lr_fn=None, master=True):
        if not torch.is_tensor(lr) and lr < 0 or weight_decay < 0 or not 0 <= momentum <= 1 or not eps > 0:
            raise ValueError("lr and weight_decay may not be negative, momentum is in [0, 1], eps above 0")
        if not 0 <= ns_steps <= 100:
            raise ValueError("ns_steps is 0 to 100")
        if adjust_lr_fn not in (None, "original", "match_rms_adamw"):
            raise ValueError("adjust_lr_fn is original (also None) or match_rms_adamw")
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, ns_coefficients=ns_coefficients, eps=eps,
                                      ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn, master=master))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()   # (what is refused is not stepped either)
                raise ValueError(f"Muon is for matrices, a parameter is {tuple(p.shape)}")

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault("master", True)

    def _state_of(self, p, group, capturing):
        s = self.state[p]
        copied = group["master"] and p.dtype != torch.float32
        if "momentum_buffer" not in s or copied and "master" not in s:
            if capturing:
                raise RuntimeError("a captured step() begins no state: make a step with the same gradients before the capture")
            if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
                raise TypeError(f"parameters are float32, bfloat16 or float16, not {p.dtype}")
            if not p.is_contiguous():
                raise ValueError("parameters are updated in place and have to be contiguous")
            if "momentum_buffer" not in s:
                s["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            if copied:
                s["master"] = p.detach().float()
        return s

    @torch.no_grad()
    def step(self, closure=None):
        """One update of every parameter that has a gradient, a call per type and device."""
        from . import ops
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        for group in self.param_groups:
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise TypeError("gradients have to be dense")
                s = self._state_of(p, group, capturing)
                calls.setdefault((p.device, p.dtype, p.grad.dtype, "master" in s), []).append((p, s))
            for (_, _, _, copies), members in calls.items():
                ps, ss = zip(*members)
                ops.muon_step([p.detach() for p in ps], [p.grad for p in ps], [s["momentum_buffer"] for s in ss], group["lr"], group["momentum"],
                              group["nesterov"], group["weight_decay"], group["ns_coefficients"], group["eps"], group["ns_steps"],
                              group["adjust_lr_fn"] or "original", [s["master"] for s in ss] if copies else None)
        return loss

    def load_state_dict(self, state_dict):
        """As the base class, but buffers are float32, those of 16-bit parameters too."""
        super().load_state_dict(state_dict)
        names = chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        for name, p in zip(names, (p for g in self.param_groups for p in g["params"])):
            if name in state_dict["state"]:
                self.state[p] = {k: v.detach().to(p.device, torch.float32, copy=True).contiguous() if torch.is_tensor(v) else v for k, v in state_dict["state"][name].items()}
