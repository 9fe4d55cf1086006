"""Layer norm over the last axis, forward and backward (K6).

``layer_norm`` is the operator under autograd; ``layer_norm_forward`` and
``layer_norm_backward`` are its two directions for code that keeps its own tape.
x is any shape [..., cols] in f32, f16 or bf16; weight and bias, each optional,
are vectors of its type.  Statistics and sums are f32.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import layers_oracle as oracle
from . import lib as _lib
from .activation8 import TYPES, Activation8, ld, lines, matrix, padded_rows, parameter, same, shaped, stream_of, type_of
from .select import _FLOAT, _ptr


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias, rstd = (variance + eps)^-1/2; mean and rstd are f32, of
    x's shape without its last axis."""
    return _forward(x, weight, bias, eps, False)


def _forward(x, weight, bias, eps, padded: bool):
    """``padded``: y of two axes, its rows on 16-byte boundaries."""
    code = type_of(x, "layer_norm")
    m = matrix(x)
    rows, cols = m.shape
    if x.size(-1) == 0:
        raise ValueError("layer_norm: the last axis is empty")
    weight = parameter(x, "weight", weight, cols)
    bias = parameter(x, "bias", bias, cols)
    if not m.is_cuda:
        y, mean, rstd = oracle.norm_forward(m, weight, bias, eps)
        return y.view(x.shape), mean.view(x.shape[:-1]), rstd.view(x.shape[:-1])
    y = padded_rows(x, rows, cols) if padded else torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    mean = x.new_empty(rows, dtype=_FLOAT)
    rstd = torch.empty_like(mean)
    if rows:
        err = _lib.calls().gtk_k6_norm_forward(code, m.data_ptr(), ld(m), _ptr(weight), _ptr(bias), y.data_ptr(), ld(y) if padded else cols,
                                               mean.data_ptr(), rstd.data_ptr(), rows, cols, eps, stream_of(m))
        if err:
            _lib.check(err, "gtk_k6_norm_forward")
    if x.dim() == 2:
        return y, mean, rstd
    return y, mean.view(x.shape[:-1]), rstd.view(x.shape[:-1])


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: Optional[torch.Tensor] = None,
                        add: Optional[torch.Tensor] = None,
                        want_parameters: bool = True) -> Tuple[torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dweight, dbias) from the forward pass's x, mean and rstd.  ``add``, of x's shape, is added to dx: the
    gradient that reaches x past the norm."""
    code = type_of(x, "layer_norm")
    m, g = matrix(x), matrix(dy)
    rows, cols = m.shape
    if dy.shape != x.shape:
        raise ValueError("the gradient has shape %s, x %s" % (tuple(dy.shape), tuple(x.shape)))
    if x.size(-1) == 0:
        raise ValueError("layer_norm: the last axis is empty")
    weight = parameter(x, "weight", weight, cols)
    same(x, dy=dy, add=add)
    if add is not None:
        shaped("add", add, *x.shape)
        add = matrix(add)
    if mean.numel() != rows or rstd.numel() != rows or mean.device != x.device or rstd.device != x.device:
        raise ValueError("mean and rstd are the forward pass's, one value for each of %d rows" % rows)
    if not m.is_cuda:
        dx, dw, db = oracle.norm_backward(g, m, mean.reshape(-1), rstd.reshape(-1), weight, add)
        return (dx.view(x.shape), dw, db) if want_parameters else (dx.view(x.shape), None, None)
    if mean.dtype is not _FLOAT or rstd.dtype is not _FLOAT:
        raise TypeError("mean and rstd are float32")
    dx = torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    dw = db = partial = None
    if want_parameters:
        dw = x.new_empty(cols)
        db = torch.empty_like(dw)
        partial = x.new_empty(min(lines("gtk_k6_norm_lines"), max(rows, 2)), 2 * cols, dtype=_FLOAT)
    if rows == 0:
        if want_parameters:
            dw.zero_()
            db.zero_()
        return dx, dw, db
    mean, rstd = mean.contiguous(), rstd.contiguous()
    err = _lib.calls().gtk_k6_norm_backward(code, g.data_ptr(), ld(g), m.data_ptr(), ld(m), None, 0, mean.data_ptr(), rstd.data_ptr(), _ptr(weight), None,
                                            _ptr(add), 0 if add is None else ld(add), dx.data_ptr(), _ptr(dw), _ptr(db), None, 0, None,
                                            _ptr(partial), rows, cols, stream_of(m))
    if err:
        _lib.check(err, "gtk_k6_norm_backward")
    return dx, dw, db


MOST_IN_BLOCK = 16384   # columns


def norm_backward_in_block(da: torch.Tensor, x, mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, dy: torch.Tensor):
    """(dx, dweight, dbias, a, dysum) over CUDA matrices of up to ``MOST_IN_BLOCK`` columns, for a block's backward pass: x
    may be codes; dx is with dy, the gradient that goes past the norm, of which dysum is the sum over the rows; a, the
    norm's output, is made again, its rows on 16-byte boundaries."""
    codes = type(x) is Activation8
    m = x.q if codes else x
    rows, cols = da.shape
    dx = da.new_empty(rows, cols)
    a = padded_rows(da, rows, cols)
    dw = da.new_empty(cols)
    db, dysum = torch.empty_like(dw), torch.empty_like(dw)
    partial = da.new_empty(min(lines("gtk_k6_norm_lines"), max(rows, 2)), 3 * cols, dtype=_FLOAT)
    err = _lib.calls().gtk_k6_norm_backward(TYPES[da.dtype], da.data_ptr(), ld(da), m.data_ptr(), ld(m), x.e.data_ptr() if codes else None,
                                            ld(x.e) if codes else 0, mean.data_ptr(), rstd.data_ptr(), weight.data_ptr(), bias.data_ptr(),
                                            dy.data_ptr(), ld(dy), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), a.data_ptr(), ld(a),
                                            dysum.data_ptr(), partial.data_ptr(), rows, cols, stream_of(da))
    if err:
        _lib.check(err, "gtk_k6_norm_backward")
    return dx, dw, db, a, dysum


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight = ctx.saved_tensors
        parameters = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dw, db = layer_norm_backward(dy, x, mean, rstd, weight, want_parameters=parameters)
        return dx, dw if ctx.needs_input_grad[1] else None, db if ctx.needs_input_grad[2] else None, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(variance + eps) * weight + bias over the last axis, under autograd."""
    return _LayerNorm.apply(x, weight, bias, eps)
