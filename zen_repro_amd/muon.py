"""The optimiser behind the exchange: momentum, orthogonalised by Newton-Schulz steps, for the matrices among a model's
parameters.  It takes the gradients where SparseCommHook (or any other all-reduce) leaves them."""
import math

import torch

from .update import COEFFICIENTS, momentum_update, orthogonal_step

_MOST_ELEMENTS = 1 << 27  # of updates that wait for their shape's call


class Muon(torch.optim.Optimizer):
    """weight = (1 - lr * weight_decay) * weight - lr * scale * O(u), with u the (Nesterov) momentum of the gradient and O its
    orthogonalisation.

    params        the layers' matrices: parameters with two dimensions, fp32 or bf16 or fp16 (embeddings, the output head and
                  everything else: any other optimiser)
    lr            about the RMS that an update's elements get, relative to `scale`
    momentum, nesterov, weight_decay, steps, coefficients, eps   see momentum_update and orthogonal_step
    match_rms     a number r: scale = r * sqrt(max(rows, cols)), which gives every update's elements an RMS of about
                  r * lr whatever the matrix' shape; None: scale = sqrt(max(1, rows / cols))
    precision     of the orthogonalisation (see orthogonal_step; default bfloat16).  The momentum hands the update on in
                  bfloat16 for bfloat16, else in float32: only its direction counts, and a small gradient is below
                  fp16's range
    The momentum is kept in fp32.  Parameters of one shape go through the orthogonalisation together."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5,
                 coefficients=COEFFICIENTS, eps=1e-7, match_rms=None, precision=torch.bfloat16):
        if lr < 0 or weight_decay < 0 or momentum < 0:
            raise ValueError("Muon: lr, momentum and weight_decay must not be negative")
        if precision not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError("Muon: precision must be float32, bfloat16 or float16")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps, match_rms=match_rms, precision=precision))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        if any(p.dim() != 2 for p in self.param_groups[-1]["params"]):
            self.param_groups.pop()
            raise ValueError("Muon: parameters have two dimensions; give the others to another optimiser")

    def load_state_dict(self, state_dict):
        """torch's gives every state its parameter's type; the momentum stays fp32."""
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        own = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(saved, own):
            momentum = state_dict["state"].get(i, {}).get("momentum")
            if momentum is not None:
                self.state[p]["momentum"] = momentum.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            alike = {}
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("Muon: sparse gradients are not supported")
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                handed_on = torch.bfloat16 if group["precision"] == torch.bfloat16 else torch.float32
                u = momentum_update(state["momentum"], p.grad.contiguous(), group["momentum"], group["nesterov"],
                                    dtype=handed_on)
                key = (p.shape, p.dtype, p.device)
                waiting = alike.setdefault(key, ([], []))
                waiting[0].append(p)
                waiting[1].append(u)
                if len(waiting[0]) * p.numel() >= _MOST_ELEMENTS:
                    self._apply(group, *alike.pop(key))
            for weights, updates in alike.values():
                self._apply(group, weights, updates)
        return loss

    def _apply(self, group, weights, updates):
        rows, cols = weights[0].shape
        if group["match_rms"] is not None:
            scale = group["match_rms"] * math.sqrt(max(rows, cols))
        else:
            scale = math.sqrt(max(1.0, rows / cols))
        orthogonal_step(weights, updates, group["lr"], group["weight_decay"], scale, group["steps"],
                        group["coefficients"], group["eps"], group["precision"])
