"""The feed-forward block of a residual network over sequences (K6, K7, K8 together).

    y = x + W2 act(W1 norm(x) + b1) + b2

``feed_forward`` computes it and what its backward pass reads: x, the norm's mean
and rstd, and z, the activation's input; with ``bits=8`` x and z are kept as
``Activation8``, 2.06 bytes a row and column of each together.  The norm's output and the
hidden layer are made again from them in the backward pass.  Of that one
(``feed_forward_backward``) the product dy W2 multiplies by the activation's slope,
makes the hidden layer again and sums b1's gradient in its epilogue.

In the 16-bit types what goes from one product to the next is rounded to the type, as the
tensor cores' operand: the norm's output, the hidden layer, dz and dz W1.  In bf16 the biases'
gradients are then 1.7e-3 off (relative norm, against 64 bits: their own rounding), y and dx
2.0e-3, dw2 2.3e-3, dw1 and the norm's gradients 2.9e-3, three roundings in a row; with fewer,
operands would have two pieces and a product be two.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import layers_oracle as oracle
from .activation8 import Activation8, act_of, bits_of, colsum, matrix, padded_rows, parameter, same, shaped, stream_of, type_of
from .layer_norm import MOST_IN_BLOCK, layer_norm_backward, norm_backward_in_block
from .layer_norm import _forward as _norm_forward
from .linear import _check, _forward, normed, operands, pairs_for, product
from .select import _FLOAT


def _norm_given(weight, bias) -> None:
    if weight is None or bias is None:
        raise ValueError("feed_forward: the norm has a weight and a bias")


class FeedForwardKept(NamedTuple):
    """What the forward pass keeps for the backward pass."""
    x: Union[torch.Tensor, Activation8]
    mean: torch.Tensor
    rstd: torch.Tensor
    z: Union[torch.Tensor, Activation8]


def feed_forward(x: torch.Tensor, norm_weight: torch.Tensor, norm_bias: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor, w2: torch.Tensor,
                 b2: torch.Tensor, activation: str = "gelu", eps: float = 1e-5, bits: int = 0,
                 keep: bool = True) -> Tuple[torch.Tensor, Optional[FeedForwardKept]]:
    """(y, kept); w1 is [hidden, dim], w2 [dim, hidden]."""
    bits_of(bits)
    if act_of(activation) == 0:
        raise ValueError("feed_forward: without an activation the two products are one")
    _check(x, w1, "feed_forward")
    shaped("w2", w2, w1.size(1), w1.size(0))
    _norm_given(norm_weight, norm_bias)
    m = matrix(x)
    a, mean, rstd = _norm_forward(m, norm_weight, norm_bias, eps, True)   # operands of the next product, where they lie
    h, z = _forward(a, w1, b1, activation, None, keep, bits, True)
    y, _ = _forward(h, w2, b2, "none", m, False, 0, False)
    if x.dim() != 2:
        y, mean, rstd = y.view(x.shape), mean.view(x.shape[:-1]), rstd.view(x.shape[:-1])
    if not keep:
        return y, None
    return y, FeedForwardKept(Activation8.keep(x) if bits else x, mean, rstd, z)


def feed_forward_backward(dy: torch.Tensor, kept: FeedForwardKept, norm_weight: torch.Tensor, norm_bias: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor,
                          activation: str = "gelu", need: Tuple[bool, ...] = (True,) * 7):
    """(dx, dnorm_weight, dnorm_bias, dw1, db1, dw2, db2), each None where ``need`` says so; what only they take is left out."""
    type_of(dy, "feed_forward")
    code = act_of(activation)
    if code == 0:
        raise ValueError("feed_forward: without an activation the two products are one")
    x, mean, rstd, z = kept
    hidden, dim = w1.shape
    shape = tuple(dy.shape)
    shaped("w2", w2, dim, hidden)
    _norm_given(norm_weight, norm_bias)
    norm_weight = parameter(dy, "norm_weight", norm_weight, dim)
    norm_bias = parameter(dy, "norm_bias", norm_bias, dim)
    if tuple(x.shape) != shape or shape[-1] != dim:
        raise ValueError("the gradient has shape %s, x %s, w1 %s" % (shape, tuple(x.shape), tuple(w1.shape)))
    same(dy, x=x, z=z, w1=w1, w2=w2)
    g = matrix(dy)
    rows = g.size(0)
    z = z if isinstance(z, Activation8) else matrix(z)
    if (tuple(z.q.shape) if isinstance(z, Activation8) else tuple(z.shape)) != (rows, hidden):
        raise ValueError("z has shape %s instead of %s" % (tuple(z.shape), (rows, hidden)))
    if mean.numel() != rows or rstd.numel() != rows or mean.device != dy.device or rstd.device != dy.device:
        raise ValueError("mean and rstd are the forward pass's, one value for each of %d rows" % rows)
    if len(need) != 7:
        raise ValueError("need has %d entries instead of 7" % len(need))
    if not g.is_cuda:
        got = _backward_plain(g, FeedForwardKept(x, mean.reshape(-1), rstd.reshape(-1), z), norm_weight, norm_bias, w1, w2, activation, shape)
        return tuple(v if n else None for v, n in zip(got, need))
    if mean.dtype is not _FLOAT or rstd.dtype is not _FLOAT:
        raise TypeError("mean and rstd are float32")
    new = dy.new_empty
    if rows == 0:
        zeros = (new(shape), *(new(n).zero_() for n in (dim, dim, (hidden, dim), hidden, (dim, hidden), dim)))
        return tuple(v if n else None for v, n in zip(zeros, need))
    stream = stream_of(g)
    mean, rstd = mean.contiguous(), rstd.contiguous()
    pairs = pairs_for(dy.dtype, True, rows, hidden, dim)
    through_norm, need_w1, need_b1, need_w2, need_b2 = any(need[:3]), *need[3:]
    dx = dg = db = dw1 = db1 = dw2 = db2 = a = None
    if through_norm or need_w1 or need_b1 or need_w2:
        # dz = (dy W2) act'(z) and h = act(z) again, both in the product's epilogue (W2's gradient alone takes h from there, too)
        dz, h = padded_rows(g, rows, hidden), padded_rows(g, rows, hidden) if need_w2 else None
        db1 = new(hidden) if need_b1 else None
        go, w2o = operands(pairs, (g, 1), (matrix(w2), 0))
        product(rows, hidden, dim, go, False, w2o, True, dz, stream, activation=code, slope=True, z=z, h=h, db=db1)
        del w2o
        if need_w2:
            dw2 = new(dim, hidden)
            if pairs:
                go, ho = operands(True, (g, 0), (h, 0))
            else:
                ho, = operands(False, (h, 0))
            product(dim, hidden, rows, go, True, ho, True, dw2, stream)
            del ho
        del h, go
    if through_norm or need_w1:
        specs = [(dz, 1), (matrix(w1), 0)] if through_norm else [] if pairs else [(dz, 0)]   # (pieces of dz do both ways, pairs one)
        if pairs and need_w1:
            specs.append((dz, 0))
        made = operands(pairs, *specs)
        zt = made[-1] if pairs or not through_norm else made[0]
    xm = x if isinstance(x, Activation8) else matrix(x)
    if through_norm:
        da = new(rows, dim)
        product(rows, dim, hidden, made[0], False, made[1], True, da, stream)
        if dim <= MOST_IN_BLOCK:   # the norm's output again and dy's sums on the way
            dx, dg, db, a, db2 = norm_backward_in_block(da, xm, mean, rstd, norm_weight, norm_bias, g)
        else:
            dx, dg, db = layer_norm_backward(da, x.restore().view(rows, dim) if isinstance(x, Activation8) else xm, mean, rstd, norm_weight, add=g,
                                             want_parameters=need[1] or need[2])
        if len(shape) != 2:
            dx = dx.view(shape)
    if need_b2 and db2 is None:
        _, db2 = colsum(g)
    if need_w1:
        if a is None:
            a = normed(xm, mean, rstd, norm_weight, norm_bias)
        dw1 = new(hidden, dim)
        ao, = operands(pairs, (a, 0))
        product(hidden, dim, rows, zt, True, ao, True, dw1, stream)
    return tuple(v if n else None for v, n in zip((dx, dg, db, dw1, db1, dw2, db2), need))


def _backward_plain(g, kept, norm_weight, norm_bias, w1, w2, activation, shape):
    def values(t):
        return oracle.values8(t.q, t.e, oracle.wide(g).dtype) if isinstance(t, Activation8) else oracle.wide(matrix(t))

    x, mean, rstd, z = values(kept.x), kept.mean, kept.rstd, values(kept.z)
    t = g.dtype
    dy = oracle.wide(g)
    dz, db1 = oracle.act_backward(dy @ oracle.wide(w2), z, activation)
    a = (x - mean[:, None]) * rstd[:, None] * oracle.wide(norm_weight) + oracle.wide(norm_bias)
    dx, dg, db = oracle.norm_backward(dz @ oracle.wide(w1), x, mean, rstd, norm_weight, dy)
    dw1, dw2 = dz.t() @ a, dy.t() @ oracle.act(activation, z)
    return tuple(v.to(t) for v in (dx.view(shape), dg, db, dw1, db1, dw2, dy.sum(0)))


class _FeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, norm_bias, w1, b1, w2, b2, activation, eps, bits, recording):
        need = recording and any(ctx.needs_input_grad)   # (which goes by the parameters, with gradients off too)
        y, kept = feed_forward(x, norm_weight, norm_bias, w1, b1, w2, b2, activation, eps, bits, need)
        if need:
            ctx.activation = activation
            xs, ctx.x = Activation8.split(kept.x)
            zs, ctx.z = Activation8.split(kept.z)
            ctx.save_for_backward(kept.mean, kept.rstd, norm_weight, norm_bias, w1, w2, *xs, *zs)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        mean, rstd, norm_weight, norm_bias, w1, w2, *rest = ctx.saved_tensors
        x, z = Activation8.join(*rest[:2], ctx.x), Activation8.join(*rest[2:], ctx.z)
        got = feed_forward_backward(dy, FeedForwardKept(x, mean, rstd, z), norm_weight, norm_bias, w1, w2, ctx.activation, tuple(ctx.needs_input_grad[:7]))
        return (*got, None, None, None, None)


def feed_forward_block(x: torch.Tensor, norm_weight: torch.Tensor, norm_bias: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor, w2: torch.Tensor,
                       b2: torch.Tensor, activation: str = "gelu", eps: float = 1e-5, bits: int = 0) -> torch.Tensor:
    """x + W2 act(W1 norm(x) + b1) + b2 under autograd; with ``bits=8`` x and the activation's input are kept in 8 bits."""
    return _FeedForward.apply(x, norm_weight, norm_bias, w1, b1, w2, b2, activation, eps, bits_of(bits), torch.is_grad_enabled())
