"""Activations kept in 8 bits between the forward and the backward pass (K7).

Blocks of 32 neighbouring columns of a row share a power of two 2^e, the least
(2^-127 at least) with max|x| <= 127 * 2^e; a value is kept as q = rint(x / 2^e),
one byte, and stands for q * 2^e.  That is 8.25 bits a value, an error of at most
half a step (max|x| / 127 at most, 1/254 of the block's largest magnitude), and a
value of 7 bits that bf16 and f32 hold exactly.  A block with a NaN or an infinity
stands for NaN throughout: what has gone wrong stays visible.  What is finite stays
finite: in the last step, 2^122, codes stop at 63.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import layers_oracle as oracle
from . import lib as _lib
from .select import _FLOAT, _ptr, _raw_stream

BLOCK = oracle.BLOCK
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # ElemType of the kernels

_lines = {}
_current_device = getattr(torch._C, "_cuda_getDevice", None)   # (torch.cuda.current_device without its checks)


def lines(name: str) -> int:
    """A constant of the library: how many lines of partial sums an entry point writes at most."""
    if name not in _lines:
        _lines[name] = int(getattr(_lib.lib(), name)())
    return _lines[name]


def type_of(t: torch.Tensor, what: str) -> int:
    """The kernels' number of a tensor's type; CPU tensors may also be f64."""
    code = TYPES.get(t.dtype)
    if code is None and not (t.device.type == "cpu" and t.dtype == torch.float64):
        raise TypeError("%s: type %s is not supported (float32, float16, bfloat16)" % (what, t.dtype))
    return -1 if code is None else code


def act_of(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError("activation %r is none of %s" % (name, ", ".join(ACTIVATIONS))) from None


def bits_of(bits: int) -> int:
    if bits not in (0, 8):
        raise ValueError("bits is 0 (kept as it is) or 8, got %r" % (bits,))
    return bits


def same(like: torch.Tensor, /, **others) -> None:
    """All given tensors (None: absent) have the type and device of ``like``."""
    for name, t in others.items():
        if t is not None and (t.dtype != like.dtype or t.device != like.device):
            raise ValueError("%s is %s on %s instead of %s on %s" % (name, t.dtype, t.device, like.dtype, like.device))


def parameter(like: torch.Tensor, name: str, t: Optional[torch.Tensor], n: int) -> Optional[torch.Tensor]:
    """A vector of n entries of the type and device of ``like``, its entries side by side; None where absent."""
    if t is None or (t.dtype is like.dtype and t.dim() == 1 and t.size(0) == n and t.is_contiguous() and t.device == like.device):
        return t
    same(like, **{name: t})
    shaped(name, t, n)
    return t.contiguous()


def shaped(name: str, t: Optional[torch.Tensor], *shape: int) -> None:
    if t is not None and tuple(t.shape) != shape:
        raise ValueError("%s has shape %s instead of %s" % (name, tuple(t.shape), shape))


def matrix(t: torch.Tensor) -> torch.Tensor:
    """t as [rows, cols] with neighbouring columns side by side; a copy only where strides allow no view."""
    if t.dim() == 2:
        if t.is_contiguous() or t.stride(1) == 1 or t.size(1) == 1:
            return t
    elif t.dim() == 0:
        raise ValueError("a scalar has no last axis")
    m = t.reshape(-1, t.size(-1)) if t.size(-1) else t.reshape(math.prod(t.shape[:-1]), 0)
    return m if m.stride(1) == 1 or m.size(1) == 1 else m.contiguous()


def ld(m: torch.Tensor) -> int:
    """Elements from one row to the next; of a single row, whose stride says nothing, its own length."""
    return m.stride(0) if m.size(0) > 1 else m.size(1)


def padded_rows(like: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """An uninitialised matrix whose rows lie on 16-byte boundaries, so that a product's kernel reads it where it is."""
    if like.dtype is _FLOAT or cols % 8 == 0:   # (f32 operands are made anew in any case)
        return like.new_empty(rows, cols)
    return like.new_empty(rows, (cols + 7) & ~7)[:, :cols]


def stream_of(t: torch.Tensor) -> int:
    """The current stream of the tensor's device, which has to be the current one: launches go there."""
    index = t.get_device()
    if index != _current_device():
        raise ValueError("the tensors are on cuda:%d, the current device is cuda:%d" % (index, _current_device()))
    return _raw_stream(index)


def colsum(dy: torch.Tensor, activation: int = 0, z=None, want_dz: bool = False, want_sum: bool = True, padded: bool = False):
    """(dz, sum of dz over the rows) with dz = dy * act'(z), over CUDA matrices; each None where not wanted.
    ``activation``: its number; ``padded``: dz's rows lie on 16-byte boundaries."""
    rows, cols = dy.shape
    dz = padded_rows(dy, rows, cols) if padded else dy.new_empty(rows, cols) if want_dz else None   # (numbers, not a tuple: half the host time)
    db = dy.new_empty(cols) if want_sum else None
    if rows == 0 or cols == 0:
        if db is not None:
            db.zero_()
        return dz, db
    if activation == 0:
        zp, zld, e, eld = None, 0, None, 0
    elif type(z) is Activation8:
        zp, zld, e, eld = z.q.data_ptr(), ld(z.q), z.e.data_ptr(), ld(z.e)
    else:
        zp, zld, e, eld = z.data_ptr(), ld(z), None, 0
    partial = dy.new_empty(min(lines("gtk_k7_act_lines"), rows), cols, dtype=_FLOAT) if want_sum else None
    err = _lib.calls().gtk_k7_act_backward(TYPES[dy.dtype], dy.data_ptr(), ld(dy), zp, zld, e, eld, activation, _ptr(dz),
                                           0 if dz is None else ld(dz), _ptr(db),
                                           _ptr(partial), rows, cols, stream_of(dy))
    if err:
        _lib.check(err, "gtk_k7_act_backward")
    return dz, db


class Activation8:
    """A tensor kept in 8 bits: ``q`` [rows, cols] int8 codes, ``e`` [rows,
    ceil(cols / 32)] uint8 exponents plus 127, and the type and shape it had."""

    __slots__ = ("q", "e", "dtype", "shape")

    def __init__(self, q: torch.Tensor, e: torch.Tensor, dtype: torch.dtype, shape: Optional[Tuple[int, ...]] = None):
        if q.dim() != 2 or q.dtype != torch.int8 or (q.size(1) > 1 and q.stride(1) != 1):
            raise ValueError("codes are an int8 matrix with neighbouring columns side by side")
        if e.dtype != torch.uint8 or tuple(e.shape) != (q.size(0), -(-q.size(1) // BLOCK)) or (e.size(1) > 1 and e.stride(1) != 1):
            raise ValueError("exponents are a uint8 matrix, one for each row and %d columns" % BLOCK)
        if e.device != q.device:
            raise ValueError("codes are on %s, exponents on %s" % (q.device, e.device))
        shape = tuple(q.shape) if shape is None else tuple(shape)
        if not shape or shape[-1] != q.size(1) or math.prod(shape[:-1]) != q.size(0):
            raise ValueError("shape %s is not that of %d rows of %d codes" % (shape, q.size(0), q.size(1)))
        if dtype not in TYPES and not (dtype == torch.float64 and not q.is_cuda):
            raise TypeError("type %s is not supported (float32, float16, bfloat16)" % dtype)
        self.q, self.e, self.dtype, self.shape = q, e, dtype, shape

    @property
    def device(self) -> torch.device:
        return self.q.device

    @staticmethod
    def split(kept):
        """What autograd saves of a tensor, or of one kept in 8 bits: (two tensors or None, what ``join`` needs besides)."""
        return ((kept.q, kept.e), (kept.dtype, kept.shape)) if type(kept) is Activation8 else ((kept, None), None)

    @staticmethod
    def join(first, second, more):
        return first if more is None else Activation8(first, second, *more)

    @property
    def nbytes(self) -> int:
        """Bytes that are held."""
        return self.q.size(0) * (ld(self.q) + ld(self.e))

    @staticmethod
    def empty(like: torch.Tensor, rows: int, cols: int, shape: Tuple[int, ...]) -> "Activation8":
        """Uninitialised, for a tensor of the type and device of ``like``; rows are padded to whole blocks, which the
        kernels store at once."""
        blocks = -(-cols // BLOCK)
        kept = Activation8.__new__(Activation8)   # consistent by construction
        q = like.new_empty(rows, blocks * BLOCK, dtype=torch.int8)
        kept.q = q if cols == blocks * BLOCK else q[:, :cols]
        kept.e = like.new_empty(rows, blocks, dtype=torch.uint8)
        kept.dtype, kept.shape = like.dtype, shape
        return kept

    @staticmethod
    def keep(x: torch.Tensor) -> "Activation8":
        """x in 8 bits."""
        code = type_of(x, "Activation8.keep")
        m = matrix(x.detach() if x.requires_grad else x)
        if not m.is_cuda:
            q, e = oracle.keep8(m)
            return Activation8(q, e, x.dtype, x.shape)
        rows, cols = m.shape
        kept = Activation8.empty(m, rows, cols, tuple(x.shape))
        if rows and cols:
            blocks = -(-cols // BLOCK)
            err = _lib.calls().gtk_k7_keep(code, m.data_ptr(), ld(m), kept.q.data_ptr(), blocks * BLOCK, kept.e.data_ptr(), blocks, rows, cols,
                                           stream_of(m))
            if err:
                _lib.check(err, "gtk_k7_keep")
        return kept

    def restore(self) -> torch.Tensor:
        """What the codes stand for, in the type and shape that the tensor had (f16 rounds steps below 2^-24)."""
        rows, cols = self.q.shape
        if not self.q.is_cuda:
            return oracle.restore8(self.q, self.e, self.dtype).view(self.shape)
        out = self.q.new_empty(rows, cols, dtype=self.dtype)
        if rows and cols:
            err = _lib.calls().gtk_k7_restore(TYPES[self.dtype], self.q.data_ptr(), ld(self.q), self.e.data_ptr(), ld(self.e), None, None, None, None,
                                              out.data_ptr(), cols, rows, cols, stream_of(self.q))
            if err:
                _lib.check(err, "gtk_k7_restore")
        return out if len(self.shape) == 2 else out.view(self.shape)

    def backward(self, dy: torch.Tensor, activation: str) -> Tuple[torch.Tensor, torch.Tensor]:
        """The kept tensor is z, an activation's input: (dz, db) with dz = dy * act'(z), and db the sum of dz over
        all but the last axis, the gradient of a bias that was added to make z."""
        code = act_of(activation)
        if dy.shape != self.shape or dy.dtype != self.dtype or dy.device != self.q.device:
            raise ValueError("the gradient is %s %s on %s, what was kept %s %s on %s"
                             % (tuple(dy.shape), dy.dtype, dy.device, self.shape, self.dtype, self.device))
        m = matrix(dy)
        if not m.is_cuda:
            dz, db = oracle.act_backward(m, oracle.values8(self.q, self.e, oracle.wide(m).dtype), activation)
            return dz.to(dy.dtype).view(self.shape), db.to(dy.dtype)
        dz, db = colsum(m, code, self, want_dz=True)
        return dz if len(self.shape) == 2 else dz.view(self.shape), db
