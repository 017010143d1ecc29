"""Operators on torch CUDA tensors for trainers with learned buckets: layer norm, routing with a balance loss, Newton-Schulz
orthogonalisation and the Muon step.

Thin wrappers over the entry points of libtatara_b200.so that work on the caller's device tensors: they check the arguments, take
outputs and workspaces from torch's allocator and enqueue on torch's current stream of the tensors' device.  Nothing is
synchronised and nothing is kept between calls.  Wrong arguments raise `TrainerError`.  This module needs torch; the rest of the
package does not.
"""
from __future__ import annotations

import ctypes as C
import threading
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib as L
from .trainer import TrainerError

_TYPES = {torch.float32: L.TYPE_F32, torch.float16: L.TYPE_F16, torch.bfloat16: L.TYPE_BF16}


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise TrainerError(what)


def _rows(t: torch.Tensor, name: str) -> int:
    """Checks a [rows, n] tensor of a supported type with adjacent columns and returns its row stride."""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise TrainerError("%s must be a CUDA tensor" % name)
    if t.dtype not in _TYPES:
        raise TrainerError("%s must be float32, float16 or bfloat16 (got %s)" % (name, t.dtype))
    if t.dim() != 2:
        raise TrainerError("%s must have two dimensions (got %d)" % (name, t.dim()))
    rows, n = t.shape
    stride, step = t.stride()
    if n > 1 and step != 1:
        raise TrainerError("%s must have adjacent columns" % name)
    if rows <= 1:
        return n
    if stride < n:
        raise TrainerError("rows of %s overlap" % name)
    return stride


def _vector(t: Optional[torch.Tensor], name: str, like: torch.Tensor, shape: Tuple[int, ...], dtype=torch.float32) -> Optional[int]:
    """Checks a contiguous tensor beside `like` and returns its address (None for None)."""
    if t is None:
        return None
    if not (isinstance(t, torch.Tensor) and t.device == like.device):
        raise TrainerError("%s must be on %s" % (name, like.device))
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise TrainerError("%s must be a contiguous %s tensor of shape %s" % (name, dtype, tuple(shape)))
    return t.data_ptr()


# torch.cuda.current_stream() builds an object in 3 us; the handle alone costs 0.1
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_local = threading.local()


def _call(name: str, like: torch.Tensor, *args) -> None:
    """Calls an entry point with the tensors' device current, on torch's current stream of it."""
    index = like.device.index
    was = torch.cuda.current_device()
    if was != index:
        torch.cuda.set_device(index)
    try:
        err = getattr(_local, "err", None)
        if err is None:
            err = _local.err = C.create_string_buffer(256)
        rc = getattr(L.load(), name)(*args, _raw_stream(index), err, 256)
        if rc != L.TB_OK:
            raise TrainerError("%s failed (%d): %s" % (name, rc, err.value.decode("utf-8", "replace")))
    finally:
        if was != index:
            torch.cuda.set_device(was)


def _work(name: str, like: torch.Tensor, *args) -> Tuple[Optional[torch.Tensor], int]:
    """A workspace of the size that an entry point asks for, and the size (sizes that it refuses are left to the call itself)."""
    index = like.device.index
    was = torch.cuda.current_device()
    if was != index:
        torch.cuda.set_device(index)
    try:
        size = getattr(L.load(), name)(*args)
    finally:
        if was != index:
            torch.cuda.set_device(was)
    return (like.new_empty(size, dtype=torch.uint8), size) if size > 0 else (None, 0)


# ---- layer norm -------------------------------------------------------------------------------------------------------
def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                       eps: float = 1e-5, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias for every row of x [rows, n]; rstd = 1 / sqrt(variance + eps).

    x and y are float32, float16 or bfloat16 with any row stride, weight and bias float32 [n]; mean and rstd (float32 [rows]) are
    what `layer_norm_backward` takes.  `out` may be x.
    """
    xs = _rows(x, "x")
    rows, n = x.shape
    y = x.new_empty((rows, n)) if out is None else out
    ys = n if out is None else _rows(out, "out")
    _need(out is None or (out.shape == x.shape and out.dtype == x.dtype and out.device == x.device), "out must match x")
    w, b = _vector(weight, "weight", x, (n,)), _vector(bias, "bias", x, (n,))
    mean = x.new_empty(rows, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    _call("tb_layer_norm_forward", x, x.data_ptr(), xs, w, b, eps, _TYPES[x.dtype], rows, n, y.data_ptr(), ys, mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                        out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of `layer_norm_forward` from the output's gradient dy [rows, n]; dweight and dbias are float32 [n]."""
    xs, gs = _rows(x, "x"), _rows(dy, "dy")
    rows, n = x.shape
    _need(dy.shape == x.shape and dy.dtype == x.dtype and dy.device == x.device, "dy must match x")
    m, r, w = _vector(mean, "mean", x, (rows,)), _vector(rstd, "rstd", x, (rows,)), _vector(weight, "weight", x, (n,))
    dx = x.new_empty((rows, n)) if out is None else out
    ds = n if out is None else _rows(out, "out")
    _need(out is None or (out.shape == x.shape and out.dtype == x.dtype and out.device == x.device), "out must match x")
    dweight = x.new_empty(n, dtype=torch.float32)
    dbias = torch.empty_like(dweight)
    work, size = _work("tb_layer_norm_backward_workspace", x, rows, n)
    _call("tb_layer_norm_backward", x, dy.data_ptr(), gs, x.data_ptr(), xs, m, r, w, _TYPES[x.dtype], rows, n, dx.data_ptr(), ds, dweight.data_ptr(),
          dbias.data_ptr(), None if work is None else work.data_ptr(), size)
    return dx, dweight, dbias


# ---- routing ----------------------------------------------------------------------------------------------------------
class Routing(NamedTuple):
    """What `route_forward` decided; `losses` holds the balance loss and the z loss."""
    index: torch.Tensor      # int32 [rows, k], -1 where no expert was left
    gate: torch.Tensor       # float32 [rows, k]
    counts: torch.Tensor     # int32 [experts]
    rows: torch.Tensor       # int32 [1]
    prob_mean: torch.Tensor  # float32 [experts]
    losses: torch.Tensor     # float32 [2]


def _mask(mask: Optional[torch.Tensor], like: torch.Tensor, rows: int) -> Optional[int]:
    if mask is None:
        return None
    return _vector(mask, "mask", like, (rows,), torch.uint8 if mask.dtype == torch.uint8 else torch.bool)


def route_forward(logits: torch.Tensor, k: int, *, renormalise: bool = True, mask: Optional[torch.Tensor] = None) -> Routing:
    """The k largest of every row's logits [rows, experts] (ties to the lowest index) as a `Routing`.

    Gates are the softmax over the chosen (`renormalise`) or over the row.  A row whose `mask` (bool [rows]) is false, or whose logits are
    all -inf, is empty; -inf forbids a single expert.  With N rows that are not empty, c the counts and P the mean softmax over them, the
    losses are experts * sum(c / (N k) * P) and the mean squared log-sum-exp.
    """
    stride = _rows(logits, "logits")
    rows, experts = logits.shape
    m = _mask(mask, logits, rows)
    _need(1 <= k, "k must be positive")
    index, gate = logits.new_empty((rows, k), dtype=torch.int32), logits.new_empty((rows, k), dtype=torch.float32)
    counts, n = logits.new_empty(experts, dtype=torch.int32), logits.new_empty(1, dtype=torch.int32)
    mean, losses = logits.new_empty(experts, dtype=torch.float32), logits.new_empty(2, dtype=torch.float32)
    work, size = _work("tb_route_forward_workspace", logits, rows, experts)
    _call("tb_route_forward", logits, logits.data_ptr(), stride, _TYPES[logits.dtype], rows, experts, k, renormalise, m, index.data_ptr(), gate.data_ptr(),
          counts.data_ptr(), n.data_ptr(), mean.data_ptr(), losses.data_ptr(), None if work is None else work.data_ptr(), size)
    return Routing(index, gate, counts, n, mean, losses)


def route_backward(logits: torch.Tensor, routing: Routing, dgate: Optional[torch.Tensor] = None, dlosses: Optional[torch.Tensor] = None, *,
                   renormalise: bool = True, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits' gradient from the gradients of the gates (float32 [rows, k]) and of the two losses (float32 [2]); the choice and the counts
    are constants.  `renormalise` and `mask` as in the `route_forward` call that gave `routing`."""
    stride = _rows(logits, "logits")
    rows, experts = logits.shape
    _need(routing.index.dim() == 2, "routing.index must have two dimensions")
    k = routing.index.shape[1]
    m = _mask(mask, logits, rows)
    ix = _vector(routing.index, "routing.index", logits, (rows, k), torch.int32)
    g, dg = _vector(routing.gate, "routing.gate", logits, (rows, k)), _vector(dgate, "dgate", logits, (rows, k))
    c, n = _vector(routing.counts, "routing.counts", logits, (experts,), torch.int32), _vector(routing.rows, "routing.rows", logits, (1,), torch.int32)
    dl = _vector(dlosses, "dlosses", logits, (2,))
    out = logits.new_empty((rows, experts))
    _call("tb_route_backward", logits, logits.data_ptr(), stride, _TYPES[logits.dtype], rows, experts, k, renormalise, m, ix, g, dg, c, n, dl, out.data_ptr(),
          experts)
    return out


# ---- orthogonalisation ------------------------------------------------------------------------------------------------
COEFFICIENTS = (3.4445, -4.7750, 2.0315)  # of the quintic step: singular values end between 0.7 and 1.2


def _matrices(t: torch.Tensor, name: str) -> Tuple[int, int, int, int, int]:
    """Checks a [rows, cols] or [batch, rows, cols] tensor with adjacent columns; (batch, rows, cols, batch stride, row stride)."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda, "%s must be a CUDA tensor" % name)
    _need(t.dtype in _TYPES, "%s must be float32, float16 or bfloat16 (got %s)" % (name, t.dtype))
    _need(t.dim() in (2, 3), "%s must have two or three dimensions (got %d)" % (name, t.dim()))
    rows, cols = t.shape[-2:]
    batch = t.shape[0] if t.dim() == 3 else 1
    _need(rows >= 1 and cols >= 1, "%s has no elements in a matrix" % name)
    stride, step = t.stride()[-2:]
    _need(cols == 1 or step == 1, "%s must have adjacent columns" % name)
    stride = stride if rows > 1 else cols
    _need(stride >= cols, "rows of %s overlap" % name)
    return batch, rows, cols, t.stride(0) if batch > 1 else 0, stride


def orthogonalise(x: torch.Tensor, *, steps: int = 5, coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Newton-Schulz orthogonalisation of x [rows, cols] or of every matrix of x [batch, rows, cols].

    X = x / (|x| + eps), then `steps` times X = (a I + b A + c A^2) X with A = X X^T over the shorter side: singular values that are not
    tiny end near 1, the singular vectors stay.  `out` may be x.
    """
    batch, rows, cols, xb, xs = _matrices(x, "x")
    y = x.new_empty(x.shape) if out is None else out
    _need(out is None or (isinstance(out, torch.Tensor) and out.shape == x.shape and out.dtype == x.dtype and out.device == x.device), "out must match x")
    _, _, _, yb, ys = _matrices(y, "out")
    _need(len(coefficients) == 3, "three coefficients are needed")
    kind = _TYPES[x.dtype]
    work, size = _work("tb_orthogonalise_workspace", x, kind, batch, rows, cols)
    _call("tb_orthogonalise", x, x.data_ptr(), xb, xs, kind, batch, rows, cols, steps, (C.c_float * 3)(*coefficients), eps, y.data_ptr(), yb, ys,
          None if work is None else work.data_ptr(), size)
    return y


def muon_step(weight: torch.Tensor, momentum: torch.Tensor, grad: torch.Tensor, *, lr: float, beta: float = 0.95, nesterov: bool = True,
              weight_decay: float = 0.0, scale: Optional[float] = None, clip: float = float("inf"), steps: int = 5,
              coefficients: Tuple[float, float, float] = COEFFICIENTS, eps: float = 1e-7, weight_out: Optional[torch.Tensor] = None,
              momentum_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """One Muon step of weight [rows, cols] or [batch, rows, cols] (float32, contiguous); returns (weight, momentum).

    m' = beta m + grad, u = grad + beta m' (`nesterov`) or m', w' = clamp(w (1 - lr weight_decay) - lr scale orthogonalise(u), -clip, clip).
    In place unless `weight_out` / `momentum_out` are given; `scale` defaults to sqrt(max(1, rows / cols)).  grad may have any type.
    """
    batch, rows, cols, _, _ = _matrices(weight, "weight")
    shape = tuple(weight.shape)
    w, m = _vector(weight, "weight", weight, shape), _vector(momentum, "momentum", weight, shape)
    _need(isinstance(grad, torch.Tensor) and grad.dtype in _TYPES, "grad must be a float32, float16 or bfloat16 tensor")
    g = _vector(grad, "grad", weight, shape, grad.dtype)
    weight_out, momentum_out = weight if weight_out is None else weight_out, momentum if momentum_out is None else momentum_out
    wo, mo = _vector(weight_out, "weight_out", weight, shape), _vector(momentum_out, "momentum_out", weight, shape)
    if scale is None:
        scale = max(1.0, rows / cols) ** 0.5
    _need(len(coefficients) == 3, "three coefficients are needed")
    cfg = L.Muon(C.sizeof(L.Muon), steps, nesterov, *coefficients, eps, lr, beta, weight_decay, scale, clip)
    work, size = _work("tb_muon_step_workspace", weight, batch, rows, cols)
    _call("tb_muon_step", weight, C.byref(cfg), w, m, g, _TYPES[grad.dtype], batch, rows, cols, wo, mo, None if work is None else work.data_ptr(), size)
    return weight_out, momentum_out
