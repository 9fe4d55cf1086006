"""Linear layer with bias, activation and residual in the product's epilogue (K8).

``linear`` is the operator under autograd; ``linear_forward`` and
``linear_backward`` are its two directions.  y = act(x W^T + bias) + residual, x
any shape [..., inner], weight [outer, inner] as in ``nn.Linear``; f32, f16 or bf16,
one type for all.  Products are summed in f32.  f32 operands are multiplied as three
bf16 pieces a value, which keeps f32's accuracy.  In the 16-bit types the gradient
dz = dy * act'(z) is rounded to the type between the products, as their operand.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import layers_oracle as oracle
from . import lib as _lib
from .activation8 import TYPES, Activation8, act_of, bits_of, colsum, ld, matrix, parameter, same, shaped, stream_of, type_of
from .select import _FLOAT, _ptr

Kept = Union[None, torch.Tensor, Activation8]


def status() -> int:
    """0, or where in the product's kernel a wait ran out (its results are void).  Synchronises."""
    return int(_lib.lib().gtk_k8_status())


class Operand:
    """A matrix as the tensor cores read it: 16-bit pieces with rows on 16-byte boundaries."""

    __slots__ = ("at", "ld", "pieces", "stride", "held")

    def __init__(self, at, row, pieces, stride, held):
        self.at, self.ld, self.pieces, self.stride, self.held = at, row, pieces, stride, held


def operands(*sources) -> list:
    """Matrices or codes (``Activation8``), up to three, as operands.  A 16-bit matrix whose rows lie on 16-byte
    boundaries is read where it is; one launch makes all the others."""
    made, words, size = [], [], 0
    for src in sources:
        codes = type(src) is Activation8
        m = src.q if codes else src
        rows, cols = m.shape
        row = ld(m)
        f32 = src.dtype is _FLOAT
        if not codes and not f32 and row % 8 == 0 and row >= cols and m.data_ptr() % 16 == 0:
            made.append(Operand(m.data_ptr(), row, 1, 0, m))
            continue
        pitch = (cols + 7) & ~7
        pieces = 3 if f32 and not codes else 1
        kind = (2 if src.dtype is torch.float16 else 3) if codes else 0 if f32 else 1
        words += (kind, m.data_ptr(), row, src.e.data_ptr() if codes else 0, ld(src.e) if codes else 0, rows, cols, size)
        made.append(Operand(size, pitch, pieces, rows * pitch, None))
        size += pieces * rows * pitch * 2
    if words:
        src = sources[0]
        room = (src.q if type(src) is Activation8 else src).new_empty(size, dtype=torch.uint8)
        base = room.data_ptr()
        for i in range(7, len(words), 8):
            words[i] += base
        for o in made:
            if o.held is None:
                o.at, o.held = o.at + base, room
        err = _lib.calls().gtk_k7_pack(words, stream_of(room))
        if err:
            _lib.check(err, "gtk_k7_pack")
    return made


def normed_operand(src, mean, rstd, weight, bias) -> Operand:
    """The operand (v - mean) * rstd * weight + bias of a matrix or of codes."""
    codes = type(src) is Activation8
    m = src.q if codes else src
    rows, cols = m.shape
    f32 = src.dtype is _FLOAT
    pieces, pitch = 3 if f32 else 1, (cols + 7) & ~7
    out = m.new_empty((pieces, rows, pitch), dtype=torch.bfloat16 if f32 else src.dtype)
    err = _lib.calls().gtk_k7_stage(TYPES[src.dtype], m.data_ptr(), ld(m), src.e.data_ptr() if codes else None, ld(src.e) if codes else 0,
                                    mean.data_ptr(), rstd.data_ptr(), _ptr(weight), _ptr(bias), 0, 3 if f32 else 0, out.data_ptr(), pitch,
                                    rows * pitch, rows, cols, pitch, stream_of(m))
    if err:
        _lib.check(err, "gtk_k7_stage")
    return Operand(out.data_ptr(), pitch, pieces, rows * pitch, out)


def product(m: int, n: int, k: int, a: Operand, a_mn: bool, b: Operand, b_mn: bool, out: torch.Tensor, stream: int, bias=None, add=None,
            activation: int = 0, slope: bool = False, z: Kept = None, h: Optional[torch.Tensor] = None, db: Optional[torch.Tensor] = None) -> None:
    """out[m, n] = epilogue(sum_k a[m, k] b[n, k]); ``a_mn``, ``b_mn``: the operand's matrix is [k, m] or [k, n].  out and
    h are dense."""
    sums = None
    zp = zld = q = qld = e = eld = None
    if z is None:
        zld = qld = eld = 0
    elif type(z) is Activation8:
        zld = 0
        q, qld, e, eld = z.q.data_ptr(), ld(z.q) if slope else z.e.size(1) * 32, z.e.data_ptr(), ld(z.e)
    else:
        qld = eld = 0
        zp, zld = z.data_ptr(), ld(z)
    if db is not None:
        sums = out.new_empty((-(-m // 32), n), dtype=_FLOAT)
    err = _lib.calls().gtk_k8_gemm(TYPES[out.dtype], out.dtype is torch.float16, m, n, k, a.at, a.ld, a.pieces, a.stride, a_mn, b.at, b.ld, b.pieces,
                                   b.stride, b_mn, out.data_ptr(), n, _ptr(bias), _ptr(add), 0 if add is None else ld(add), activation, slope, zp,
                                   zld, q, qld, e, eld, _ptr(h), n, _ptr(sums), _ptr(db), stream)
    if err:
        _lib.check(err, "gtk_k8_gemm")


def _check(x, weight, what):
    if weight.dim() != 2:
        raise ValueError("%s: weight is a matrix [outer, inner]" % what)
    if weight.size(1) == 0 or x.shape[-1] != weight.size(1):
        raise ValueError("%s: the input's last axis has %d entries, weight is %s" % (what, x.shape[-1], tuple(weight.shape)))


def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
                   residual: Optional[torch.Tensor] = None, keep: bool = False, bits: int = 0) -> Tuple[torch.Tensor, Kept]:
    """(y, z): y = act(x W^T + bias) + residual.  With ``keep`` z is the activation's input for ``linear_backward``, in
    x's type or, with ``bits=8``, as ``Activation8``; None where there is no activation."""
    type_of(x, "linear")
    code = act_of(activation)
    if bits:
        bits_of(bits)
    _check(x, weight, "linear")
    same(x, weight=weight, residual=residual)
    outer, inner = weight.shape
    shape = (*x.shape[:-1], outer)
    bias = parameter(x, "bias", bias, outer)
    if residual is not None:
        shaped("residual", residual, *shape)
        residual = matrix(residual)
    keep = keep and code != 0
    m = matrix(x)
    rows = m.size(0)
    if not m.is_cuda:
        y, z = oracle.linear_forward(m, weight, bias, activation, residual)
        z = None if not keep else Activation8(*oracle.keep8(z), x.dtype) if bits else z.to(x.dtype)
        return y.view(shape), z
    y = x.new_empty(shape)
    z = None
    if keep:
        z = Activation8.empty(x, rows, outer, (rows, outer)) if bits else x.new_empty((rows, outer))
    if rows and outer:
        a, b = operands(m, matrix(weight))
        product(rows, outer, inner, a, False, b, False, y, stream_of(m), bias, residual, code, z=z)
    return y, z


def _gradients(dz: torch.Tensor, x, weight: torch.Tensor, need_dx: bool, need_dw: bool):
    """(dz W, dz^T x) over CUDA matrices; x may be codes, or an operand already."""
    rows, outer = dz.shape
    inner = weight.size(1)
    dx = dw = None
    if not (need_dx or need_dw):
        return dx, dw
    stream = stream_of(dz)
    made = type(x) is Operand
    a, *rest = operands(dz, *((matrix(weight),) if need_dx else ()), *((x,) if need_dw and not made else ()))
    if need_dx:
        dx = dz.new_empty((rows, inner))
        product(rows, inner, outer, a, False, rest[0], True, dx, stream)
    if need_dw:
        dw = dz.new_empty((outer, inner))
        product(outer, inner, rows, a, True, x if made else rest[-1], True, dw, stream)
    return dx, dw


def linear_backward(dy: torch.Tensor, x: Union[torch.Tensor, Activation8], weight: torch.Tensor, activation: str = "none", z: Kept = None,
                    need: Tuple[bool, bool, bool] = (True, True, True)):
    """(dx, dweight, dbias), each None where ``need`` says so, from x (which may have been kept in 8 bits) and from the
    z that ``linear_forward`` kept.  The residual's gradient is dy."""
    type_of(dy, "linear")
    code = act_of(activation)
    _check(x, weight, "linear_backward")
    outer, inner = weight.shape
    shape = tuple(x.shape)
    if tuple(dy.shape) != (*shape[:-1], outer):
        raise ValueError("the gradient has shape %s, x %s, weight %s" % (tuple(dy.shape), shape, tuple(weight.shape)))
    same(dy, weight=weight, x=x)
    g = matrix(dy)
    rows = g.size(0)
    if code:
        if z is None:
            raise ValueError("linear_backward: the activation's input z is missing")
        same(dy, z=z)
        z = z if isinstance(z, Activation8) else matrix(z)
        if (tuple(z.q.shape) if isinstance(z, Activation8) else tuple(z.shape)) != (rows, outer):
            raise ValueError("z does not have the gradient's shape")
    if not g.is_cuda:
        zv = oracle.values8(z.q, z.e, oracle.wide(dy).dtype) if isinstance(z, Activation8) else z
        dz, db = oracle.act_backward(g, zv, activation)
        xv = oracle.values8(x.q, x.e, dz.dtype) if isinstance(x, Activation8) else oracle.wide(matrix(x))
        return ((dz @ oracle.wide(weight)).to(dy.dtype).view(shape) if need[0] else None, (dz.t() @ xv).to(dy.dtype) if need[1] else None,
                db.to(dy.dtype) if need[2] else None)
    if rows == 0 or outer == 0:
        return (torch.zeros(shape, dtype=dy.dtype, device=dy.device) if need[0] else None, torch.zeros_like(weight) if need[1] else None,
                torch.zeros(outer, dtype=dy.dtype, device=dy.device) if need[2] else None)
    products = need[0] or need[1]
    db = None
    if (code and products) or need[2]:
        dz, db = colsum(g, code, z, want_dz=bool(code and products), want_sum=need[2])
        g = dz if code and products else g
    dx, dw = _gradients(g, x if isinstance(x, Activation8) or not need[1] else matrix(x), weight, need[0], need[1])
    return dx if dx is None or len(shape) == 2 else dx.view(shape), dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual, bits):
        y, z = linear_forward(x, weight, bias, activation, residual, keep=any(ctx.needs_input_grad[:3]), bits=bits)
        ctx.activation = activation
        ctx.z = z if isinstance(z, Activation8) else None
        kept = Activation8.keep(x) if bits and ctx.needs_input_grad[1] else None
        ctx.x = kept if kept is not None else x.shape if bits else None
        ctx.save_for_backward(None if bits else x, weight, None if isinstance(z, Activation8) else z)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            if x is None:   # kept in 8 bits, or not kept at all where the weight has no gradient
                x = ctx.x if isinstance(ctx.x, Activation8) else dy.new_empty(1).expand(ctx.x)
            dx, dw, db = linear_backward(dy, x, weight, ctx.activation, z if ctx.z is None else ctx.z, tuple(need[:3]))
        return dx, dw, db, None, dy if need[4] else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, bits: int = 0) -> torch.Tensor:
    """act(x W^T + bias) + residual under autograd.  With ``bits=8`` the backward pass reads x and the activation's
    input from 8-bit copies (``Activation8``), and nothing larger of them is held."""
    return _Linear.apply(x, weight, bias, activation, residual, bits_of(bits))
