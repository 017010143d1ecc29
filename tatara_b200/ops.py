"""Operators on torch CUDA tensors for trainers with learned buckets: layer norm, routing with a balance loss, Newton-Schulz
orthogonalisation and the Muon step.

Thin wrappers over the entry points of libtatara_b200.so that work on the caller's device tensors: they check the arguments, take
outputs and workspaces from torch's allocator and enqueue on torch's current stream of the tensors' device.  Nothing is
synchronised and nothing is kept between calls.  Wrong arguments raise `TrainerError`.  This module needs torch; the rest of the
package does not.
"""
from __future__ import annotations

import ctypes as C
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
    _need(isinstance(t, torch.Tensor) and t.is_cuda, "%s must be a CUDA tensor" % name)
    _need(t.dtype in _TYPES, "%s must be float32, float16 or bfloat16 (got %s)" % (name, t.dtype))
    _need(t.dim() == 2, "%s must have two dimensions (got %d)" % (name, t.dim()))
    rows, n = t.shape
    stride, step = t.stride()
    _need(n <= 1 or step == 1, "%s must have adjacent columns" % name)
    _need(rows <= 1 or stride >= n, "rows of %s overlap" % name)
    return stride if rows > 1 else max(stride, n)


def _vector(t: Optional[torch.Tensor], name: str, like: torch.Tensor, shape: Tuple[int, ...], dtype=torch.float32) -> Optional[int]:
    """Checks a contiguous tensor beside `like` and returns its address (None for None)."""
    if t is None:
        return None
    _need(isinstance(t, torch.Tensor) and t.device == like.device, "%s must be on %s" % (name, like.device))
    _need(t.dtype == dtype and t.shape == shape and t.is_contiguous(), "%s must be a contiguous %s tensor of shape %s" % (name, dtype, tuple(shape)))
    return t.data_ptr()


class _On:
    """Makes a tensor's device current where it is not."""
    __slots__ = ("was", "index")

    def __init__(self, t: torch.Tensor):
        self.index = t.device.index

    def __enter__(self):
        self.was = torch.cuda.current_device()
        if self.was != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *exc):
        if self.was != self.index:
            torch.cuda.set_device(self.was)


def _call(name: str, *args) -> None:
    err = C.create_string_buffer(256)
    rc = getattr(L.load(), name)(*args, err, 256)
    if rc != L.TB_OK:
        raise TrainerError("%s failed (%d): %s" % (name, rc, err.value.decode("utf-8", "replace")))


# ---- layer norm -------------------------------------------------------------------------------------------------------
def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *,
                       eps: float = 1e-5, out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias for every row of x [rows, n]; rstd = 1 / sqrt(variance + eps).

    x and y are float32, float16 or bfloat16 with any row stride, weight and bias float32 [n]; mean and rstd (float32 [rows]) are
    what `layer_norm_backward` takes.  `out` may be x.
    """
    xs = _rows(x, "x")
    rows, n = x.shape
    y = torch.empty((rows, n), dtype=x.dtype, device=x.device) if out is None else out
    ys = n if out is None else _rows(out, "out")
    _need(out is None or (out.shape == x.shape and out.dtype == x.dtype and out.device == x.device), "out must match x")
    w, b = _vector(weight, "weight", x, (n,)), _vector(bias, "bias", x, (n,))
    mean, rstd = torch.empty(rows, dtype=torch.float32, device=x.device), torch.empty(rows, dtype=torch.float32, device=x.device)
    with _On(x) as stream:
        _call("tb_layer_norm_forward", x.data_ptr(), xs, w, b, eps, _TYPES[x.dtype], rows, n, y.data_ptr(), ys, mean.data_ptr(), rstd.data_ptr(), stream)
    return y, mean, rstd


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None, *,
                        out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dx, dweight, dbias) of `layer_norm_forward` from the output's gradient dy [rows, n]; dweight and dbias are float32 [n]."""
    xs, gs = _rows(x, "x"), _rows(dy, "dy")
    rows, n = x.shape
    _need(dy.shape == x.shape and dy.dtype == x.dtype and dy.device == x.device, "dy must match x")
    m, r, w = _vector(mean, "mean", x, (rows,)), _vector(rstd, "rstd", x, (rows,)), _vector(weight, "weight", x, (n,))
    dx = torch.empty((rows, n), dtype=x.dtype, device=x.device) if out is None else out
    ds = n if out is None else _rows(out, "out")
    _need(out is None or (out.shape == x.shape and out.dtype == x.dtype and out.device == x.device), "out must match x")
    d = torch.empty((2, n), dtype=torch.float32, device=x.device)
    with _On(x) as stream:
        size = L.load().tb_layer_norm_backward_workspace(rows, n)
        work = torch.empty(max(size, 1), dtype=torch.uint8, device=x.device)
        p = d.data_ptr()
        _call("tb_layer_norm_backward", dy.data_ptr(), gs, x.data_ptr(), xs, m, r, w, _TYPES[x.dtype], rows, n, dx.data_ptr(), ds, p, p + 4 * n,
              work.data_ptr(), size, stream)
    return dx, d[0], d[1]


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
    dev = logits.device
    m = _mask(mask, logits, rows)
    _need(1 <= k, "k must be positive")
    index, gate = torch.empty((rows, k), dtype=torch.int32, device=dev), torch.empty((rows, k), dtype=torch.float32, device=dev)
    whole, real = torch.empty(experts + 1, dtype=torch.int32, device=dev), torch.empty(experts + 2, dtype=torch.float32, device=dev)
    with _On(logits) as stream:
        size = L.load().tb_route_forward_workspace(rows, experts)
        work = torch.empty(max(size, 1), dtype=torch.uint8, device=dev)
        c, p = whole.data_ptr(), real.data_ptr()
        _call("tb_route_forward", logits.data_ptr(), stride, _TYPES[logits.dtype], rows, experts, k, renormalise, m, index.data_ptr(), gate.data_ptr(), c,
              c + 4 * experts, p, p + 4 * experts, work.data_ptr(), size, stream)
    return Routing(index, gate, whole[:experts], whole[experts:], real[:experts], real[experts:])


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
    out = torch.empty((rows, experts), dtype=logits.dtype, device=logits.device)
    with _On(logits) as stream:
        _call("tb_route_backward", logits.data_ptr(), stride, _TYPES[logits.dtype], rows, experts, k, renormalise, m, ix, g, dg, c, n, dl, out.data_ptr(),
              experts, stream)
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
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device) if out is None else out
    _need(out is None or (isinstance(out, torch.Tensor) and out.shape == x.shape and out.dtype == x.dtype and out.device == x.device), "out must match x")
    _, _, _, yb, ys = _matrices(y, "out")
    _need(len(coefficients) == 3, "three coefficients are needed")
    kind = _TYPES[x.dtype]
    with _On(x) as stream:
        size = L.load().tb_orthogonalise_workspace(kind, batch, rows, cols)
        work = torch.empty(size, dtype=torch.uint8, device=x.device) if size > 0 else None
        _call("tb_orthogonalise", x.data_ptr(), xb, xs, kind, batch, rows, cols, steps, (C.c_float * 3)(*coefficients), eps, y.data_ptr(), yb, ys,
              None if work is None else work.data_ptr(), max(size, 0), stream)
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
    with _On(weight) as stream:
        size = L.load().tb_muon_step_workspace(batch, rows, cols)
        work = torch.empty(size, dtype=torch.uint8, device=weight.device) if size > 0 else None
        _call("tb_muon_step", C.byref(cfg), w, m, g, _TYPES[grad.dtype], batch, rows, cols, wo, mo, None if work is None else work.data_ptr(), max(size, 0), stream)
    return weight_out, momentum_out
