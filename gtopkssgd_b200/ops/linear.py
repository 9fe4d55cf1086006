"""Linear layer with bias, activation and residual in the product's epilogue (K8; K9 for few rows).

``linear`` is the operator under autograd; ``linear_forward`` and
``linear_backward`` are its two directions.  y = act(x W^T + bias) + residual, x
any shape [..., inner], weight [outer, inner] as in ``nn.Linear``; f32, f16 or bf16,
one type for all.  Products are summed in f32.  f32 operands are multiplied as three
bf16 pieces a value, which keeps f32's accuracy entry by entry (what is left out is 2^-22 of
a product's magnitude at most).  A program may choose two scaled f16 pieces, which are faster and keep it
relative to a row's largest entry only: ``PAIRS_FROM_FORWARD``.  In the 16-bit types the gradient
dz = dy * act'(z) is rounded to the type between the products, as their operand.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import settings
from . import layers_oracle as oracle
from . import lib as _lib
from .activation8 import TYPES, Activation8, act_of, bits_of, colsum, ld, matrix, padded_rows, parameter, same, shaped, stream_of, type_of
from .select import _FLOAT, _ptr

# Rows up to which K9 takes a forward pass, us on the device by K9 and by K8, whose operands have to be made first: 1500 x 6000
# in bf16 1, 8, 20 and 32 rows 7, 8, 12 and 14 against 22, in f32 12, 12, 27 and 29 against 48; and a launch less.
FEW_ROWS = 32

Kept = Union[None, torch.Tensor, Activation8]


_launched = False   # whether this process has launched a product


def status() -> int:
    """0, or where in the product's kernel a wait ran out since the status was last cleared (the results of that product,
    and what was computed from them, are void).  Of the current device.  Synchronises."""
    return int(_lib.lib().gtk_k8_status())


def check_status() -> None:
    """Raises GtopkNativeError where a wait of a product ran out.  ``DistributedOptimizer.check_status`` and the training
    loops, every so many steps, do this; synchronises, and does nothing where no product was launched."""
    where = status() if _launched else 0
    if where:
        raise _lib.GtopkNativeError("a linear layer's product: a wait ran out (code location %d); results since the last check are void" % where)


def clear_status() -> None:
    """Sets the status to 0, after its results have been thrown away.  Synchronises."""
    _lib.check(_lib.lib().gtk_k8_clear_status(), "gtk_k8_clear_status")


def rehearse_timeout(device: torch.device, limit_ms: float = 50.0) -> torch.Tensor:
    """Lets one wait run out on the device, as a product's would behind work that never ends, so that what a program does
    about it can be tried: afterwards ``status()`` is not 0 and ``check_status`` raises.  Returns what each of 32 lanes of the waiting warp was told, of
    which the first waits for something that is there: 0 for all of them, as they have to go on together."""
    global _launched
    _launched = True
    answers = torch.empty(32, dtype=torch.int32, device=device)
    _lib.check(_lib.calls().gtk_k8_rehearse_wait(int(limit_ms * 1e6), answers.data_ptr(), stream_of(answers)), "gtk_k8_rehearse_wait")
    return answers


class Operand:
    """A matrix as the tensor cores read it: 16-bit pieces with rows on 16-byte boundaries.  ``most``: the largest
    magnitudes that two f16 pieces were scaled by, else 0."""

    __slots__ = ("at", "ld", "pieces", "stride", "most", "held")

    def __init__(self, at, row, pieces, stride, most, held):
        self.at, self.ld, self.pieces, self.stride, self.most, self.held = at, row, pieces, stride, most, held


# f32 operands as two f16 pieces (three products instead of six) from this many multiplications a product on; None: never.
# A vector of an operand along the contracted axis (a row of x or W forward, a column of dz, x or W for the gradients that sum
# over it) is scaled by a power of two that takes its largest magnitude M just below 2^15, and entries below 2^-17 M lose
# bits: each is off by 2^-40 M at most, whatever its own size, and a result by that times the sum of its partners'
# magnitudes.  Where one entry of 2^30 meets a zero weight - a masked token, an unused channel - the others' products are 1e-3
# off, so that only a program that knows its entries can choose this.  It does from about 500_000_000 forward and
# 2_200_000_000 backward (whose operands are scaled by columns: two launches more, and read once more).
PAIRS_FROM_FORWARD: Optional[int] = None
PAIRS_FROM_BACKWARD: Optional[int] = None


def pairs_for(dtype: torch.dtype, backward: bool, m: int, n: int, k: int) -> bool:
    least = PAIRS_FROM_BACKWARD if backward else PAIRS_FROM_FORWARD
    return least is not None and dtype is _FLOAT and m * n * k >= least


def operands(pairs: bool, *specs) -> list:
    """Up to four matrices or codes (``Activation8``) as operands; each comes as (matrix, contracted), ``contracted`` the
    axis of it that the product sums over.  A 16-bit matrix whose rows lie on 16-byte boundaries is read where it is;
    one launch makes all the others (``pairs``: f32 as two f16 pieces)."""
    made, words, size, row_most, column_most = [], [], 0, 0, 0
    for src, contracted in specs:
        codes = type(src) is Activation8
        f32 = src.dtype is _FLOAT
        if codes and pairs:
            src, codes = src.restore().view(src.q.shape), False
        m = src.q if codes else src
        rows, cols = m.shape
        row = ld(m)
        if not codes and not f32 and row % 8 == 0 and row >= cols and m.data_ptr() % 16 == 0:
            made.append(Operand(m.data_ptr(), row, 1, 0, 0, m))
            continue
        pitch = (cols + 7) & ~7
        if codes:
            kind, pieces, scale = 2 if src.dtype is torch.float16 else 3, 1, src.e.data_ptr()
        elif not f32:
            kind, pieces, scale = 1, 1, 0
        elif not pairs:
            kind, pieces, scale = 0, 3, 0
        elif contracted == 1:
            kind, pieces, scale = 4, 2, row_most
            row_most += rows
        else:
            kind, pieces, scale = 5, 2, column_most
            column_most += cols
        words += (kind, m.data_ptr(), row, scale, ld(src.e) if codes else 0, rows, cols, size)
        made.append(Operand(size, pitch, pieces, rows * pitch, scale if kind >= 4 else 0, (m, kind)))
        size += pieces * rows * pitch * 2
    if words:
        src = specs[0][0]
        like = src.q if type(src) is Activation8 else src
        room = like.new_empty(size + 4 * row_most, dtype=torch.uint8)
        zeros = like.new_zeros(column_most, dtype=torch.int32) if column_most else None
        base, rows_at, columns_at = room.data_ptr(), room.data_ptr() + size, zeros.data_ptr() if column_most else 0
        for i in range(0, len(words), 8):
            words[i + 7] += base
            if words[i] == 4:
                words[i + 3] = rows_at + 4 * words[i + 3]
            elif words[i] == 5:
                words[i + 3] = columns_at + 4 * words[i + 3]
        err = _lib.calls().gtk_k7_pack(words, stream_of(room))
        if err:
            _lib.check(err, "gtk_k7_pack")
        for o in made:
            if type(o.held) is tuple:
                kind = o.held[1]
                o.at += base
                if kind >= 4:
                    o.most = (rows_at if kind == 4 else columns_at) + 4 * o.most
                o.held = (room, zeros)
    return made


def normed(src, mean, rstd, weight, bias) -> torch.Tensor:
    """The matrix (v - mean) * rstd * weight + bias of a matrix or of codes."""
    codes = type(src) is Activation8
    m = src.q if codes else src
    rows, cols = m.shape
    out = m.new_empty(rows, cols, dtype=src.dtype)
    err = _lib.calls().gtk_k7_restore(TYPES[src.dtype], m.data_ptr(), ld(m), src.e.data_ptr() if codes else None, ld(src.e) if codes else 0,
                                      mean.data_ptr(), rstd.data_ptr(), _ptr(weight), _ptr(bias), out.data_ptr(), cols, rows, cols, stream_of(m))
    if err:
        _lib.check(err, "gtk_k7_restore")
    return out


def product(m: int, n: int, k: int, a: Operand, a_mn: bool, b: Operand, b_mn: bool, out: torch.Tensor, stream: int, bias=None, add=None,
            activation: int = 0, slope: bool = False, z: Kept = None, h: Optional[torch.Tensor] = None, db: Optional[torch.Tensor] = None) -> None:
    """out[m, n] = epilogue(sum_k a[m, k] b[n, k]); ``a_mn``, ``b_mn``: the operand's matrix is [k, m] or [k, n]."""
    global _launched
    _launched = True
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
        sums = out.new_empty(-(-m // 32), n, dtype=_FLOAT)
    err = _lib.calls().gtk_k8_gemm(TYPES[out.dtype], out.dtype is torch.float16 or a.pieces == 2, m, n, k, a.at, a.ld, a.pieces, a.stride, a_mn,
                                   a.most or None, b.at, b.ld, b.pieces, b.stride, b_mn, b.most or None, out.data_ptr(), ld(out), _ptr(bias), _ptr(add),
                                   0 if add is None else ld(add), activation, slope, zp, zld, q, qld, e, eld, _ptr(h), 0 if h is None else ld(h),
                                   _ptr(sums), _ptr(db), int(settings.WAIT_LIMIT_MS * 1e6), stream)
    if err:
        _lib.check(err, "gtk_k8_gemm")


def _check(x, weight, what):
    if weight.dim() != 2:
        raise ValueError("%s: weight is a matrix [outer, inner]" % what)
    inner = weight.size(1)
    if not x.shape:
        raise ValueError("%s: a scalar has no last axis" % what)
    if inner == 0 or x.shape[-1] != inner:
        raise ValueError("%s: the input's last axis has %d entries, weight is %s" % (what, x.shape[-1], tuple(weight.shape)))


def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
                   residual: Optional[torch.Tensor] = None, keep: bool = False, bits: int = 0) -> Tuple[torch.Tensor, Kept]:
    """(y, z): y = act(x W^T + bias) + residual.  With ``keep`` z is the activation's input for ``linear_backward``, in
    x's type or, with ``bits=8``, as ``Activation8``; None where there is no activation."""
    return _forward(x, weight, bias, activation, residual, keep, bits, False)


def _forward(x, weight, bias, activation, residual, keep, bits, padded: bool):
    """``padded``: y of two axes, its rows on 16-byte boundaries."""
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
    y = padded_rows(x, rows, outer) if padded else x.new_empty(rows, outer)
    z = None
    if keep:
        z = Activation8.empty(x, rows, outer, (rows, outer)) if bits else x.new_empty(rows, outer)
    if rows == 0 or outer == 0:
        return y if x.dim() == 2 else y.view(shape), z
    if rows <= FEW_ROWS:   # K9 reads x and W where they are
        w = matrix(weight)
        zp = q = e = None
        qld = eld = 0
        if z is not None:
            if bits:
                q, qld, e, eld = z.q.data_ptr(), z.e.size(1) * 32, z.e.data_ptr(), z.e.size(1)
            else:
                zp = z.data_ptr()
        err = _lib.calls().gtk_k9_few_rows(TYPES[x.dtype], m.data_ptr(), ld(m), w.data_ptr(), ld(w), rows, outer, inner, y.data_ptr(), ld(y), _ptr(bias),
                                           _ptr(residual), 0 if residual is None else ld(residual), code, zp, q, qld, e, eld, stream_of(m))
        if err:
            _lib.check(err, "gtk_k9_few_rows")
    else:
        a, b = operands(pairs_for(x.dtype, False, rows, outer, inner), (m, 1), (matrix(weight), 1))
        product(rows, outer, inner, a, False, b, False, y, stream_of(m), bias, residual, code, z=z)
    return y if x.dim() == 2 else y.view(shape), z


def _gradients(dz: torch.Tensor, x, weight: torch.Tensor, need_dx: bool, need_dw: bool):
    """(dz W, dz^T x) over CUDA matrices; x may be codes."""
    rows, outer = dz.shape
    inner = weight.size(1)
    dx = dw = None
    if not (need_dx or need_dw):
        return dx, dw
    stream = stream_of(dz)
    pairs = pairs_for(dz.dtype, True, rows, outer, inner)
    specs = [(dz, 1)] if need_dx or not pairs else []
    if need_dx:
        specs.append((matrix(weight), 0))
    if need_dw and pairs:
        specs.append((dz, 0))
    if need_dw:
        specs.append((x, 0))
    made = operands(pairs, *specs)
    if need_dx:
        dx = dz.new_empty(rows, inner)
        product(rows, inner, outer, made[0], False, made[1], True, dx, stream)
    if need_dw:
        dw = dz.new_empty(outer, inner)
        a, b = made[-2] if pairs else made[0], made[-1]
        product(outer, inner, rows, a, True, b, True, dw, stream)
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
        dz, db = colsum(g, code, z, want_dz=bool(code and products), want_sum=need[2], padded=bool(code and products))
        g = dz if code and products else g
    dx, dw = _gradients(g, x if isinstance(x, Activation8) or not need[1] else matrix(x), weight, need[0], need[1])
    return dx if dx is None or len(shape) == 2 else dx.view(shape), dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, activation, residual, bits, recording):
        # needs_input_grad goes by the parameters, with gradients off too; in here they always are
        y, z = linear_forward(x, weight, bias, activation, residual, keep=recording and any(ctx.needs_input_grad[:3]), bits=bits)
        if not recording:
            return y
        ctx.activation, ctx.shape = activation, x.shape
        if not ctx.needs_input_grad[1]:
            x = None
        elif bits:   # all that is kept goes through autograd, which lets go of it behind the backward pass
            x = Activation8.keep(x)
        xs, ctx.x = Activation8.split(x)
        zs, ctx.z = Activation8.split(z)
        ctx.save_for_backward(weight, *xs, *zs)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight, *kept = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if any(need[:3]):
            x, z = Activation8.join(*kept[:2], ctx.x), Activation8.join(*kept[2:], ctx.z)
            if x is None:   # not kept where the weight has no gradient
                x = dy.new_empty(1).expand(ctx.shape)
            dx, dw, db = linear_backward(dy, x, weight, ctx.activation, z, tuple(need[:3]))
        return dx, dw, db, None, dy if need[4] else None, None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None, bits: int = 0) -> torch.Tensor:
    """act(x W^T + bias) + residual under autograd.  With ``bits=8`` the backward pass reads x and the activation's
    input from 8-bit copies (``Activation8``), and nothing larger of them is held."""
    return _Linear.apply(x, weight, bias, activation, residual, bits_of(bits), torch.is_grad_enabled())
