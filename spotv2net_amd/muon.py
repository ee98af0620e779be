"""Orthogonalised weight updates on hand-written gfx950 kernels.

``orthogonalize(g)`` maps a matrix (or each matrix of a stack) to one with the
same singular vectors and singular values near 1 by Newton-Schulz steps: X = g /
max(|g|_F, eps), then ``steps`` times S = X Xt, X <- a X + (b S + c S S) X.

``muon_step`` updates a list of weight matrices in place from their gradients
and momenta with it, all of them in the same launches; ``Muon`` is the optimiser
over it.  ``train.TrainStep(optimizer="muon")`` trains a model with it, beside
Adam for what is not a matrix between hidden features (the reference trains
everything with Adam, 5_train_SpotV2Net.py:127).
"""
from __future__ import annotations

import math
from typing import Sequence, Tuple

import torch

from . import library  # noqa: F401  (registers torch.ops.sv2n.muon_step)

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _check_device(what: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"spotv2net_amd runs {what} only on a ROCm GPU (got a "
                           f"{t.device.type} tensor); there is no CPU fallback")


def orthogonalize(g: torch.Tensor, steps: int = 5,
                  coefficients: Tuple[float, float, float] = COEFFICIENTS,
                  eps: float = 1e-7) -> torch.Tensor:
    """The Newton-Schulz orthogonalisation of ``g`` ([rows, cols], or a stack
    [k, rows, cols] of matrices that are each their own); float32, bfloat16 or
    float16, sides up to 16,384.  For every type the result is as accurate as one of
    f32 products, measured over the whole matrix, and rounded once.  (Rows or columns
    under about 2^-16 of the norm keep fewer bits of their own and under 2^-39 none,
    unless ``steps`` are so many that they could grow to a visible part: include/sv2n.h.)
    Not differentiable."""
    _check_device("orthogonalize", g)
    a, b, c = coefficients
    return torch.ops.sv2n.orthogonalize(g.detach(), steps, a, b, c, eps)


def lr_scale(rows: int, cols: int, adjust: str = "original") -> float:
    """The factor of the learning rate for a [rows, cols] weight: "original":
    sqrt(max(1, rows / cols)); "match_rms_adamw": 0.2 sqrt(max(rows, cols)), an
    update of about the root mean square of an Adam step."""
    if adjust == "original":
        return math.sqrt(max(1.0, rows / cols)) if cols else 1.0
    if adjust == "match_rms_adamw":
        return 0.2 * math.sqrt(max(rows, cols))
    raise ValueError(f'adjust_lr is "original" or "match_rms_adamw", got {adjust!r}')


@torch.no_grad()
def muon_step(weights: Sequence[torch.Tensor], grads: Sequence[torch.Tensor],
              momenta: Sequence[torch.Tensor], lr: float, momentum: float = 0.95,
              nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
              coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7,
              adjust_lr: str = "original") -> None:
    """One step over float32 weight matrices, in place (weights and momenta):
    m <- beta m + (1 - beta) g;  u = (1 - beta) g + beta m (nesterov) or m;
    w <- (1 - lr weight_decay) w - lr lr_scale(w) orthogonalize(u)."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    for t in weights:
        _check_device("muon_step", t)
        if t.dim() != 2:
            raise ValueError(f"muon_step updates matrices, got shape {tuple(t.shape)}")
    if not weights:
        return
    a, b, c = coefficients
    torch.ops.sv2n.muon_step(weights, grads, momenta,
                             [lr_scale(w.shape[0], w.shape[1], adjust_lr) for w in weights], lr,
                             momentum, nesterov, weight_decay, steps, a, b, c, eps)
    # the kernels write through raw pointers: autograd learns of it here
    # (inference tensors have no version to raise)
    torch.autograd.graph.increment_version(
        [t for t in weights + momenta if not t.is_inference()])


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates for weight matrices (2-D float32
    parameters); everything else belongs to another optimiser.  One ``step`` is
    ``2 + 3 steps`` launches per 16 matrices of a parameter group (sides past about
    1,200: up to twice as many; thin matrices beside large ones: ``1 + steps`` more;
    small ones alone: fewer), without a host synchronisation, and can be captured into
    a graph after a first step outside of it."""

    def __init__(self, params, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, coefficients: Tuple[float, float, float] = COEFFICIENTS,
                 eps: float = 1e-7, steps: int = 5, adjust_lr: str = "original"):
        if lr < 0.0 or weight_decay < 0.0 or not 0.0 <= momentum < 1.0:
            raise ValueError(f"Muon: lr {lr}, weight_decay {weight_decay}, momentum {momentum}")
        lr_scale(1, 1, adjust_lr)  # refuses an unknown rule
        super().__init__(params, dict(lr=lr, weight_decay=weight_decay, momentum=momentum,
                                      nesterov=nesterov, coefficients=tuple(coefficients), eps=eps,
                                      steps=steps, adjust_lr=adjust_lr))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() != 2 or p.dtype != torch.float32:
                    raise ValueError("Muon takes 2-D float32 parameters, got "
                                     f"{tuple(p.shape)} {p.dtype}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            ws = [p for p in group["params"] if p.grad is not None]
            for p in ws:
                if "momentum_buffer" not in self.state[p]:
                    if p.is_cuda and torch.cuda.is_current_stream_capturing():
                        # its zeros would be part of the graph, and of every replay
                        raise RuntimeError("Muon: run one step before capturing one (the "
                                           "momentum is allocated by the first)")
                    self.state[p]["momentum_buffer"] = torch.zeros_like(
                        p, memory_format=torch.contiguous_format)
            muon_step(ws, [p.grad for p in ws], [self.state[p]["momentum_buffer"] for p in ws],
                      lr=group["lr"], momentum=group["momentum"], nesterov=group["nesterov"],
                      weight_decay=group["weight_decay"], steps=group["steps"],
                      coefficients=group["coefficients"], eps=group["eps"],
                      adjust_lr=group["adjust_lr"])
        return loss
