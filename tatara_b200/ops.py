"""Operators on torch CUDA tensors for trainers with learned buckets: layer norm, routing with a balance loss, Newton-Schulz
orthogonalisation and the Muon step.

The functions check their arguments, take outputs and workspaces from torch's allocator and enqueue kernels of libtatara_b200.so on torch's current
stream of the tensors' device (csrc/torch_ops.cpp).  Nothing is synchronised and nothing is kept between calls.  Wrong arguments raise
`TrainerError`.  Small results of one call (mean and rstd; dweight and dbias; a routing's counts, rows, prob_mean and losses) are parts of one
allocation: clone what is to outlive the others by long.  Gradients are what the *_backward functions return; torch's automatic differentiation
does not see these calls, but it refuses to use what it saved of a tensor that one of them has written since (`out`, or a Muon step's weight and momentum).  This module needs torch; the rest of the package does not.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .trainer import TrainerError

_lib.load()
try:
    from . import _ops
except ImportError as e:
    raise ImportError("tatara_b200: the torch binding _ops.so is missing or was built for another torch (%s); build it with `python -m tatara_b200.build`. "
                      "There is no fallback." % e) from e
_ops.set_error(TrainerError)


# ---- layer norm -------------------------------------------------------------------------------------------------------
def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                       eps: float = 1e-5, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias for every row of x [rows, n]; rstd = 1 / sqrt(variance + eps).

    x and y are float32, float16 or bfloat16 with any row stride, weight and bias float32 [n]; mean and rstd (float32 [rows]) are
    what `layer_norm_backward` takes.  `out` may be x.
    """
    return _ops.layer_norm_forward(x, weight, bias, eps, out)


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                        out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of `layer_norm_forward` from the output's gradient dy [rows, n]; dweight and dbias are float32 [n].  `out` may be dy
    or x."""
    return _ops.layer_norm_backward(dy, x, mean, rstd, weight, out)


# ---- routing ----------------------------------------------------------------------------------------------------------
class Routing(NamedTuple):
    """What `route_forward` decided; `losses` holds the balance loss and the z loss."""
    index: torch.Tensor      # int32 [rows, k], -1 where no expert was left
    gate: torch.Tensor       # float32 [rows, k]
    counts: torch.Tensor     # int32 [experts]
    rows: torch.Tensor       # int32 [1]
    prob_mean: torch.Tensor  # float32 [experts]
    losses: torch.Tensor     # float32 [2]


def route_forward(logits: torch.Tensor, k: int, *, renormalise: bool = True, mask: Optional[torch.Tensor] = None) -> Routing:
    """The k largest of every row's logits [rows, experts] (ties to the lowest index) as a `Routing`.

    Gates are the softmax over the chosen (`renormalise`) or over the row.  A row whose `mask` (bool [rows]) is false, or whose logits are
    all -inf, is empty; -inf forbids a single expert.  With N rows that are not empty, c the counts and P the mean softmax over them, the
    losses are experts * sum(c / (N k) * P) and the mean squared log-sum-exp.  At most 1024 experts and 16 choices.
    """
    return Routing._make(_ops.route_forward(logits, k, renormalise, mask))


def route_backward(logits: torch.Tensor, routing: Routing, dgate: Optional[torch.Tensor] = None, dlosses: Optional[torch.Tensor] = None, *,
                   renormalise: bool = True, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits' gradient from the gradients of the gates (float32 [rows, k]) and of the two losses (float32 [2]); the choice and the counts
    are constants.  `renormalise` and `mask` as in the `route_forward` call that gave `routing`."""
    return _ops.route_backward(logits, routing.index, routing.gate, routing.counts, routing.rows, dgate, dlosses, renormalise, mask)


# ---- orthogonalisation ------------------------------------------------------------------------------------------------
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of the quintic step: singular values end between 0.7 and 1.2


def orthogonalise(x: torch.Tensor, *, steps: int = 5, coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of x [rows, cols] or of every matrix of x [batch, rows, cols].

    X = x / (|x| + eps), then `steps` times X = (a I + b A + c A^2) X with A = X X^T over the shorter side: singular values that are not
    tiny end near 1, the singular vectors stay.  `out` may be x.  With a shorter side above 64, float32 and float16 matrices are multiplied from 22-bit operands,
    bfloat16 ones from 11-bit operands at half to a third of the time: 1e-3 of the result beside its own rounding of 1.7e-3.  Give float32 for more.
    """
    return _ops.orthogonalise(x, steps, coefficients, eps, out)


def muon_step(weight: torch.Tensor, momentum: torch.Tensor, grad: torch.Tensor, *, lr: float, beta: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.0, scale: Optional[float] = None, clip: float = float("inf"), steps: int = 5,
              coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7, weight_out: Optional[torch.Tensor] = None,
              momentum_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One Muon step of weight [rows, cols] or [batch, rows, cols] (float32, contiguous); returns (weight, momentum).

    m' = beta m + grad, u = grad + beta m' (`nesterov`) or m', w' = clamp(w (1 - lr weight_decay) - lr scale orthogonalise(u), -clip, clip).
    In place unless `weight_out` / `momentum_out` are given; `scale` defaults to sqrt(max(1, rows / cols)).  grad may have any type.
    """
    return _ops.muon_step(weight, momentum, grad, weight_out, momentum_out, steps, nesterov, coefficients, eps, lr, beta, weight_decay, scale, clip)
