"""Optimiser of projection matrices: momentum whose update is orthogonalised by Newton-Schulz products.

:func:`orthogonalize` runs ``m3_orthogonalize`` on CUDA and the same products in float32 on the CPU;
:class:`Muon` is the optimiser on top of it.
"""

from __future__ import annotations

import math

import torch

from . import _ext

# x' = a x + b (x x^T) x + c (x x^T)^2 x: a steep odd polynomial whose iterates carry every singular
# value in (0, 1] to about 1 (0.7 to 1.2) in five steps. They, the Nesterov form and the scale of Muon's
# update are those published with it (Keller Jordan and others, 2024)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def _orthogonalize_torch(x, steps, coefficients):
    a, b, c = coefficients
    x = x.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    norm = torch.linalg.matrix_norm(x, keepdim=True)
    x = x / torch.where(norm == 0, torch.ones_like(norm), norm)
    for _ in range(steps):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


@torch.no_grad()
def orthogonalize(update: torch.Tensor, steps: int = 5, *, coefficients=COEFFICIENTS,
                  out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The Newton-Schulz iterate of ``update`` (``[rows, cols]`` or ``[..., rows, cols]``), its
    singular values carried towards 1; zero matrices stay zero. The result is ``out_dtype``; on CUDA
    the products are taken in 16 bits with float32 sums, whatever the types, so that a float32 result
    too is within about 1e-3 of its norm, and entries of an iterate or of ``x x^T`` must stay below 255
    (coefficients that carry singular values past 15 do not). No derivative: forward mode is refused there."""
    if update.dim() < 2:
        raise ValueError("update must be a matrix or a stack of matrices")
    if not 0 <= steps <= 64:
        raise ValueError("steps must be in [0, 64]")
    if len(coefficients) != 3:
        raise ValueError("coefficients are three numbers a, b, c")
    if update.numel() == 0:
        return update.to(out_dtype)
    if not update.is_cuda:
        return _orthogonalize_torch(update, steps, coefficients).to(out_dtype).contiguous()
    if _ext.has_tangent(update):
        raise ValueError("orthogonalize has no forward-mode derivative on CUDA")
    if update.dtype not in _FLOATS or out_dtype not in _FLOATS:
        raise TypeError(f"unsupported dtypes {update.dtype} -> {out_dtype}")
    stack = update.unsqueeze(0) if update.dim() == 2 else update.flatten(0, -3)
    return _ext.orthogonalize(stack, steps, coefficients, out_dtype).view(update.shape)


def _wide(p: torch.Tensor) -> torch.dtype:
    return torch.promote_types(p.dtype, torch.float32)


class Muon(torch.optim.Optimizer):
    """Momentum SGD whose update of every matrix is orthogonalised, for the 2-D weights of hidden
    layers (``in_proj`` / ``out_proj``); embeddings, norms and vectors belong to another optimiser.

        m <- momentum m + grad;  u = orthogonalize(grad + momentum m if nesterov else m)
        w <- w (1 - lr weight_decay) - lr scale u,   scale = sqrt(max(1, rows / cols))

    Matrices of one shape, dtype and device are orthogonalised as one stack. The momentum is held in
    float32 for 16-bit weights too, and u is formed from it there.
    """

    def __init__(self, params, lr: float = 0.02, *, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5) -> None:
        if lr < 0.0 or not 0.0 <= momentum < 1.0 or weight_decay < 0.0:
            raise ValueError("lr and weight_decay must not be negative, momentum must be in [0, 1)")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps))

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2:
                self.param_groups.pop()
                raise ValueError(f"Muon updates matrices; got a parameter of shape {tuple(p.shape)}")

    def load_state_dict(self, state_dict) -> None:
        super().load_state_dict(state_dict)  # which casts the momentum to its weight's type
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(saved, (p for group in self.param_groups for p in group["params"])):
            held = self.state.get(p, {}).get("momentum")
            if held is not None and held.dtype != _wide(p):
                self.state[p]["momentum"] = state_dict["state"][i]["momentum"].to(p.device, _wide(p), copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            stacks: dict[tuple, list] = {}
            for p in group["params"]:
                if p.grad is not None:
                    stacks.setdefault((p.shape, p.dtype, p.device), []).append(p)
            for (shape, _, _), params in stacks.items():
                grads = [p.grad.to(_wide(p)) for p in params]
                for p in params:
                    if "momentum" not in self.state[p]:
                        self.state[p]["momentum"] = torch.zeros_like(p, dtype=_wide(p))
                buffers = [self.state[p]["momentum"] for p in params]
                torch._foreach_mul_(buffers, group["momentum"])
                torch._foreach_add_(buffers, grads)
                updates = torch._foreach_add(grads, buffers, alpha=group["momentum"]) if group["nesterov"] else buffers
                directions = orthogonalize(torch.stack(updates), group["steps"])
                if group["weight_decay"]:
                    torch._foreach_mul_(params, 1.0 - group["lr"] * group["weight_decay"])
                scale = math.sqrt(max(1.0, shape[0] / max(1, shape[1])))
                torch._foreach_add_(params, [d.to(p.dtype) for d, p in zip(directions.unbind(0), params)],
                                    alpha=-group["lr"] * scale)
        return loss
