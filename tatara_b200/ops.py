"""Operators on torch CUDA tensors for trainers with learned buckets: layer norm, root-mean-square norm on a residual stream, routing with a balance loss, rows sorted
by expert and back, rows of a table by token, Newton-Schulz orthogonalisation and the Muon step.

The functions check their arguments, take outputs and workspaces from torch's allocator and enqueue kernels of libtatara_b200.so on torch's current
stream of the tensors' device (csrc/torch_ops.cpp).  Nothing is synchronised and nothing is kept between calls.  Wrong arguments raise
`TrainerError`.  Small results of one call (mean and rstd; dweight and dbias; a routing's counts, rows, prob_mean and losses; an order's three; a residual stream's h and rstd) are parts of one
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


# ---- root-mean-square norm ----------------------------------------------------------------------------------------------
def rms_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     out: Optional[torch.Tensor] = None, residual_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, h, rstd): h = x + residual and y = h * rstd * weight for every row of x [rows, n]; rstd = 1 / sqrt(mean(h^2) + eps).

    x, residual, y and h are of one type (float32, float16 or bfloat16) with any row strides, weight float32 [n].  y is the norm of the 32-bit sum, h the sum
    rounded to the type (x itself without a residual): the residual of the next layer.  h and rstd (float32 [rows]) are what `rms_norm_backward` takes.  `out` and
    `residual_out` may be x or residual, not both the same.  Where y is written over x without a residual, h is that memory too and no longer what `rms_norm_backward` takes.  Without `eps`, a
    row of zeros is NaN.
    """
    return _ops.rms_norm_forward(x, weight, residual, eps, out, residual_out)


def rms_norm_quantised(x: torch.Tensor, weight: Optional[torch.Tensor] = None, *, residual: Optional[torch.Tensor] = None, eps: float = 1e-6,
                       group: Optional[int] = None, residual_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(q, scale, h, rstd): `rms_norm_forward` with y ~ q * scale in 8 bits.

    q is float8_e4m3fn [rows, n], scale float32 [rows, ceil(n / group)]: the largest |y| of a row's group of 32, 64, 128 or (None) all columns over 448, at least
    2^-126.  The backward pass is `rms_norm_backward`, as if y had not been rounded.  A group whose y holds an infinity or a NaN is NaN throughout.
    """
    return _ops.rms_norm_quantised(x, weight, residual, eps, group, residual_out)


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None, *, dresidual: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight) of `rms_norm_forward` from the gradients dy of y and `dresidual` of h (what later layers send back along the residual stream).  dx [rows, n] is the
    gradient of x and of the residual alike, dweight float32 [n].  `out` may be dy, h or dresidual."""
    return _ops.rms_norm_backward(dy, h, rstd, weight, dresidual, out)


# ---- rows by expert -----------------------------------------------------------------------------------------------------
class Order(NamedTuple):
    """Where the choices of a router go when they are sorted by expert."""
    position: torch.Tensor  # int32 [rows, k]: the place of every choice, -1 where there is none
    source: torch.Tensor    # int32 [places]: the choice r * k + j of every place, -1 where there is none
    offsets: torch.Tensor   # int32 [experts + 1]: expert e has the places offsets[e] to offsets[e + 1]


def expert_order(index: torch.Tensor, experts: int, *, align: int = 1) -> Order:
    """The choices index [rows, k] (int32, as in a `Routing`) sorted by expert, an expert's by row and then choice.

    Anything outside [0, experts) is no choice.  Every expert has a multiple of `align` places, as tiles of a product need them.  The number of places is that of the worst
    case, so that nothing waits for the device: rows * k without `align`; those behind offsets[experts] are left over.  At most 1024 experts and 16 choices.
    """
    return Order._make(_ops.expert_order(index, experts, align))


def dispatch_forward(x: torch.Tensor, order: Order) -> torch.Tensor:
    """[places, n]: the row x[r] at every place of its choices, zeros at places without a choice.  x [rows, n] is float32, float16 or bfloat16."""
    return _ops.dispatch_forward(x, order.position, order.source)


def dispatch_backward(dy: torch.Tensor, order: Order) -> torch.Tensor:
    """The gradient of `dispatch_forward`'s x from that of its places: every row's are added up."""
    return _ops.combine_forward(dy, order.position, order.source, None)


def combine_forward(y: torch.Tensor, order: Order, gate: torch.Tensor) -> torch.Tensor:
    """[rows, n]: out[r] = sum of gate[r, j] * y[position[r, j]] over the choices of row r that have a place; y [places, n], gate float32 [rows, k]."""
    if gate is None:
        raise TrainerError("gate must be a tensor")
    return _ops.combine_forward(y, order.position, order.source, gate)


def combine_backward(dout: torch.Tensor, y: torch.Tensor, order: Order, gate: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dy, dgate) of `combine_forward` from the gradient dout [rows, n] of its result: dy [places, n], zeros at places without a choice, and dgate float32 [rows, k], 0
    where a choice has no place."""
    return _ops.combine_backward(dout, y, order.position, order.source, gate)


# ---- rows by token ------------------------------------------------------------------------------------------------------
def embedding_forward(tokens: torch.Tensor, table: torch.Tensor, *, scale: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """scale * table[tokens]: tokens int32 or int64 of any shape, table [rows, n] float32, float16 or bfloat16.  A token outside the table (-1 for padding) has a row of zeros."""
    return _ops.embedding_forward(tokens, table, scale, out)


def embedding_backward(dy: torch.Tensor, tokens: torch.Tensor, rows: int, *, scale: float = 1.0, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The gradient [rows, n] of `embedding_forward`'s table from dy (tokens' shape and n): scale * the sum of dy over the tokens of every row, zeros where there are none.

    Sums are 32 bits wide in an order that depends on the tokens alone.  `dtype` is that of dy (the default) or float32.
    """
    if dtype not in (None, torch.float32, getattr(dy, "dtype", None)):
        raise TrainerError("dtype must be that of dy or float32")
    return _ops.embedding_backward(dy, tokens, rows, scale, dtype == torch.float32)


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
