"""The feed-forward operators' kernels against the formulas in 64 bits.

Tolerances are bounds, not fits.  With u the unit roundoff of the result's type
(2^-24, 2^-11, 2^-8) and S the sum of the magnitudes of what is added up for an
entry, a result is at most u * |result| + c * 2^-24 * S away: the rounding where it
is stored, and f32 sums.  c = 64 covers sums in registers, across lanes and lines
(chains of at most some 40 additions here); tensor-core sums cut instead of
rounding, once per 16 of the contracted length (f32: once per 16 of each 256), so a
product has c = 2 * (length / 16 + 24) at most.
"""
import math

import pytest
import torch
import torch.nn.functional as F

from gtopkssgd_b200.ops import layers_oracle as oracle
from gtopkssgd_b200.ops.activation8 import Activation8
from gtopkssgd_b200.ops.feed_forward import FeedForwardKept, feed_forward, feed_forward_backward, feed_forward_block
from gtopkssgd_b200.ops.layer_norm import layer_norm, layer_norm_backward, layer_norm_forward
from gtopkssgd_b200.ops.linear import linear, linear_backward, linear_forward, status

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.float16, torch.bfloat16]
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}   # the smallest step of a type
EPS32 = 2.0 ** -24


def _randn(*shape, dtype=torch.float32, scale=1.0, seed=None):
    gen = torch.Generator(device=DEV).manual_seed(sum(shape) * 31 + len(shape) if seed is None else seed)
    return (torch.randn(*shape, device=DEV, generator=gen) * scale).to(dtype)


def _within(got, want, bound, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs()
    limit = U[got.dtype] * want.abs() + bound + LEAST[got.dtype]
    assert torch.all((off <= limit) | (got == want.to(got.dtype))), "%s: %g over a bound of %g" % (what, float((off - limit).max()), float(limit.flatten()[int((off - limit).argmax())]))


def _c(length, dtype):
    return 2 * EPS32 * ((256 if dtype == torch.float32 else length) / 16 + length / 256 + 24)


# -- layer norm ---------------------------------------------------------------------
def _check_norm(x, w, b, dy, add=None, eps=1e-5):
    y, mean, rstd = layer_norm_forward(x, w, b, eps)
    X = x.double()
    m = X.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((X - m) ** 2).mean(-1, keepdim=True) + eps)
    xh = (X - m) * r
    W = torch.ones(x.size(-1), dtype=torch.float64, device=DEV) if w is None else w.double()
    B = torch.zeros_like(W) if b is None else b.double()
    size = X.abs().mean(-1, keepdim=True)
    # the mean is off by c * eps32 * mean|x|, which moves xh by that times rstd
    mean_off = 64 * EPS32 * size
    _within(mean, m.squeeze(-1), mean_off.squeeze(-1), "mean")
    rel = 64 * EPS32 * (1 + (mean_off * r) ** 2 * 64)
    assert torch.all((rstd.double() - r.squeeze(-1)).abs() <= (rel * r).squeeze(-1) + EPS32 * r.squeeze(-1)), "rstd"
    _within(y, xh * W + B, 64 * EPS32 * (((X - m).abs() + X.abs()) * r * W.abs() + B.abs()) + mean_off * r * W.abs(), "y")
    # backward, from the statistics that the forward pass gave
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w, add=add)
    m, r = mean.double().unsqueeze(-1), rstd.double().unsqueeze(-1)
    xh, G = (X - m) * r, dy.double()
    t = G * W
    want = r * (t - t.mean(-1, keepdim=True) - xh * (t * xh).mean(-1, keepdim=True)) + (0 if add is None else add.double())
    xh_off = 4 * EPS32 * (X.abs() + m.abs()) * r + 4 * EPS32 * xh.abs()    # of xh, from the subtraction
    bound = 64 * EPS32 * r * (t.abs() + t.abs().mean(-1, keepdim=True) + xh.abs() * (t * xh).abs().mean(-1, keepdim=True)) \
        + r * (xh_off * (t * xh).abs().mean(-1, keepdim=True) + xh.abs() * (t.abs() * xh_off).mean(-1, keepdim=True))
    if add is not None:
        bound = bound + 2 * EPS32 * add.double().abs()
    _within(dx, want, bound, "dx")
    G, xh, xh_off = (v.expand(x.shape).reshape(-1, x.size(-1)) for v in (G, xh, xh_off))
    _within(dw, (G * xh).sum(0), 64 * EPS32 * (G * xh).abs().sum(0) + (G.abs() * xh_off).sum(0), "dw")
    _within(db, G.sum(0), 64 * EPS32 * G.abs().sum(0), "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 2), (2, 33), (3, 1000), (20, 1500), (7, 1021), (300, 256), (5, 4096), (700, 1500), (6, 8192), (3, 8200),
                                       (4, 12000), (2, 16384), (3, 20001), (1, 9000), (1, 16384), (1, 30000), (8, 1500), (33, 64)])
def test_layer_norm(dtype, rows, cols):
    x = _randn(rows, cols, dtype=dtype) * _randn(cols, dtype=dtype).abs() + _randn(cols, dtype=dtype)
    _check_norm(x, _randn(cols, dtype=dtype, seed=1), _randn(cols, dtype=dtype, seed=2), _randn(rows, cols, dtype=dtype, seed=3),
                _randn(rows, cols, dtype=dtype, seed=4) if rows % 2 else None)


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_without_parameters_and_with_strides(dtype):
    _check_norm(_randn(9, 40, dtype=dtype), None, None, _randn(9, 40, dtype=dtype, seed=1))
    _check_norm(_randn(9, 40, dtype=dtype), _randn(40, dtype=dtype), None, _randn(9, 40, dtype=dtype, seed=1))
    wide = _randn(9, 100, dtype=dtype)
    _check_norm(wide[:, 3:67], None, None, _randn(9, 128, dtype=dtype, seed=1)[:, 64:])      # rows apart, off the boundary
    _check_norm(wide[:, ::2], None, None, _randn(9, 50, dtype=dtype, seed=1))
    _check_norm(wide[::3, :64], None, None, _randn(3, 64, dtype=dtype, seed=1))
    _check_norm(_randn(4, 5, 32, dtype=dtype).transpose(0, 1), None, None, _randn(5, 4, 32, dtype=dtype, seed=1))
    _check_norm(_randn(1, 64, dtype=dtype).expand(6, 64), None, None, _randn(6, 64, dtype=dtype, seed=1))   # rows at the same place
    _check_norm(_randn(200, dtype=dtype)[1:], None, None, _randn(199, dtype=dtype, seed=1))  # one axis


def test_layer_norm_special_rows():
    """Constant rows, rows far from zero, NaN and infinity only in their own row."""
    x = _randn(6, 1500)
    x[1] = 3.0
    x[2] += 1e4
    x[3, 7] = math.nan
    x[4, 9] = math.inf
    y, mean, rstd = layer_norm_forward(x)
    assert torch.equal(y[1], torch.zeros(1500, device=DEV)) and float(rstd[1]) == pytest.approx(1e-5 ** -0.5, rel=1e-6)
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[4]).any()
    for row in (0, 2, 5):
        want = F.layer_norm(x[row].double(), (1500,))
        assert torch.allclose(y[row].double(), want, atol=2e-3 if row == 2 else 1e-5)
    dx, dw, db = layer_norm_backward(torch.ones_like(x), x, mean, rstd)
    assert torch.isfinite(dx[[0, 1, 2, 5]]).all() and torch.isnan(dx[3]).all() and torch.isnan(dw[7])
    empty = torch.empty(0, 1500, device=DEV)
    y, mean, rstd = layer_norm_forward(empty)
    dx, dw, db = layer_norm_backward(empty, empty, mean, rstd)
    assert y.shape == dx.shape == (0, 1500) and not dw.any() and not db.any()


@pytest.mark.parametrize("rows,cols", [(700, 1500), (37, 1021), (20, 64), (3, 9000)])
@pytest.mark.parametrize("ratio", [100.0, 1e4])
def test_layer_norm_gradients_of_rows_far_from_zero(rows, cols, ratio):
    """Means of ``ratio`` standard deviations.  From the statistics given, x - mean is off by a rounding of its own size and
    so is its product with rstd: xh to 3 * 2^-24 of xh, and no part of it goes by the mean's size."""
    x = _randn(rows, cols) + ratio
    dy, w = _randn(rows, cols, seed=1), _randn(cols, seed=2)
    _, mean, rstd = layer_norm_forward(x, w)
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w)
    r = rstd.double()[:, None]
    xh, G, W = (x.double() - mean.double()[:, None]) * r, dy.double(), w.double()
    t = G * W
    want = r * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
    _within(dx, want, 70 * EPS32 * r * (t.abs() + t.abs().mean(1, keepdim=True) + xh.abs() * (t * xh).abs().mean(1, keepdim=True)), "dx")
    _within(dw, (G * xh).sum(0), 70 * EPS32 * (G * xh).abs().sum(0), "dw")
    # in a block: the norm's output that is made again is the forward pass's
    p = [w, _randn(cols, seed=3), _randn(24, cols, scale=cols ** -0.5, seed=4), _randn(24, seed=5), _randn(cols, 24, scale=0.2, seed=6), _randn(cols, seed=7)]
    kept = feed_forward(x, *p)[1]
    got = feed_forward_backward(dy, kept, *p[:3], p[4])
    dz = (G @ p[4].double()) * oracle.act_slope("gelu", kept.z.double())
    da = dz @ p[2].double()
    for have, want, what in ((got[1], (da * xh).sum(0), "dg"), (got[3], dz.t() @ (xh * W + p[1].double()), "dw1")):
        assert float((have.double() - want).norm()) <= 2e-6 * float(want.norm()), what


# -- 8 bits ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (3, 32), (5, 33), (20, 1500), (7, 1021), (700, 600), (2, 12004)])
def test_codes_equal_the_plain_ones(dtype, rows, cols):
    x = (_randn(rows, cols) * torch.exp(3 * _randn(rows, 1, seed=5))).to(dtype)
    for m in (x, F.pad(x, (1, 3))[:, 1:-3]):
        kept = Activation8.keep(m)
        q, e = oracle.keep8(m)
        assert torch.equal(kept.q, q) and torch.equal(kept.e, e)
        back, want = kept.restore(), oracle.restore8(q, e, dtype)
        assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back[~want.isnan()], want[~want.isnan()])


def test_codes_of_special_values():
    tiny, big = 2.0 ** -149, torch.finfo(torch.float32).max
    rows = [[0.0], [tiny], [2.0 ** -126, 2.0 ** -127], [2.0 ** -121 * 127 / 64, 1e-38], [127.0, 0.5, 1.5], [127.0 + 2 ** -17, 1.0, 3.0], [big, -big, 1.0],
            [math.inf, 1.0], [1.0, -math.inf], [math.nan], [-0.0, 1.0], [254.0, 3.0, -3.0]]
    x = torch.zeros(len(rows), 70, device=DEV)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r)
        x[i, 64:64 + len(r)] = torch.tensor(r)       # a block of six columns
    kept = Activation8.keep(x)
    q, e = oracle.keep8(x.cpu())
    assert torch.equal(kept.q.cpu(), q) and torch.equal(kept.e.cpu(), e)
    back = kept.restore()
    assert torch.equal(back.isnan().cpu(), oracle.values8(q, e).isnan())
    assert torch.equal(back.nan_to_num(7.0).cpu(), oracle.values8(q, e).nan_to_num(7.0))
    assert torch.isfinite(back[6]).all() and back[7:10, :32].isnan().all() and (back[7:10, 32:64] == 0).all()
    half = torch.full((2, 40), 65504.0, device=DEV, dtype=torch.float16)
    assert torch.equal(Activation8.keep(half).restore(), half)
    assert Activation8.keep(torch.empty(0, 40, device=DEV)).restore().shape == (0, 40)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (20, 1500), (333, 1021), (3000, 96)])
def test_gradient_through_a_kept_activation(dtype, name, rows, cols):
    kept = Activation8.keep(_randn(rows, cols, dtype=dtype, scale=2.0))
    dy = _randn(rows, cols, dtype=dtype, seed=9)
    dz, db = kept.backward(dy, name)
    z = oracle.values8(kept.q, kept.e, torch.float64)
    want = dy.double() * oracle.act_slope(name, z)
    # slopes are f32 expressions of magnitudes up to 1 + |z|, with erf, exp and tanh good to a few units
    off = 16 * EPS32 * dy.double().abs() * (1 + z.abs())
    _within(dz, want, off, "dz")
    _within(db, want.sum(0), 64 * EPS32 * want.abs().sum(0) + off.sum(0), "db")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cols", [64, 70, 72, 96])
def test_codes_of_large_values(dtype, cols):
    """Every step up to the last, 2^122, whatever the width of a thread's loads: restored values are the codes' exactly, and
    what is finite stays finite on the way back too (a slope of a large positive value is 1, of a negative one 0)."""
    steps = [90, 103, 104, 105, 106, 110, 116, 121, 122]
    x = _randn(len(steps), cols).to(dtype)
    for i, e in enumerate(steps):
        x[i] = (x[i] / x[i].abs().max() * 2.0 ** 6 * 0.96).double().mul(2.0 ** e).to(dtype)   # 61.4 * 2^e is the largest
        x[i, 1], x[i, cols - 1] = 0.0, 2.0 ** e
    kept = Activation8.keep(x)
    q, e = oracle.keep8(x.cpu())
    assert torch.equal(kept.q.cpu(), q) and torch.equal(kept.e.cpu(), e) and int(kept.e.max()) >= 121 + 127
    back = kept.restore()
    assert torch.equal(back.cpu(), oracle.restore8(q, e, dtype)) and back.isfinite().all()
    dy = _randn(len(steps), cols, dtype=dtype, seed=2)
    z = oracle.values8(kept.q, kept.e, torch.float64)
    for name in ("none", "relu", "gelu", "silu"):
        dz, db = kept.backward(dy, name)
        want = dy.double() * oracle.act_slope(name, z)
        _within(dz, want, 16 * EPS32 * dy.double().abs(), name)
        _within(db, want.sum(0), 80 * EPS32 * dy.double().abs().sum(0), name)
    # x from codes under the norm of a block's backward pass, at steps whose squares f32 does not hold
    rows, hidden = len(steps), 40
    mean = z.mean(1).float()
    rstd = (1 / (z - mean.double()[:, None]).square().mean(1).sqrt()).clamp(min=2.0 ** -126).float()
    small = _randn(rows, hidden, dtype=dtype, seed=3)
    p = [_randn(cols, dtype=dtype, seed=4), _randn(cols, dtype=dtype, seed=5), _randn(hidden, cols, dtype=dtype, seed=6), _randn(cols, hidden, dtype=dtype, seed=7)]
    got = feed_forward_backward(dy, FeedForwardKept(kept, mean, rstd, Activation8.keep(small)), *p, "silu")
    g, b, w1, w2 = (t.double() for t in p)
    h = oracle.values8(*oracle.keep8(small), torch.float64)
    dz = (dy.double() @ w2) * oracle.act_slope("silu", h)
    xh = (z - mean.double()[:, None]) * rstd.double()[:, None]
    da = dz @ w1
    limit = max(1e-5, 8 * U[dtype])
    for have, want, what in zip(got[1:4], ((da * xh).sum(0), da.sum(0), dz.t() @ (xh * g + b)), ("dg", "db", "dw1")):
        assert float((have.double() - want).norm()) <= limit * float(want.norm()), what
    assert got[0].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_of_large_values(dtype, name):
    """1 and 0, also where the square of z is past f32's range."""
    from gtopkssgd_b200.ops.activation8 import ACTIVATIONS, colsum
    z = torch.tensor([1e19, 2e19, 1e25, 3e38, 400.0], device=DEV).repeat_interleave(32)      # a block of 32 each
    z = torch.stack([z, -z]).to(dtype)
    dy = _randn(2, 160, dtype=dtype)
    want = torch.stack([dy[0], torch.zeros_like(dy[1])])
    for got in (Activation8.keep(z).backward(dy, name)[0], colsum(dy, ACTIVATIONS[name], z, want_dz=True)[0]):
        assert torch.equal(got, want)


# -- linear ---------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 40, 33), (3, 7, 5), (20, 1500, 600), (64, 64, 128), (129, 65, 257), (128, 1000, 64), (515, 1001, 130), (300, 2000, 96),
          (1, 4096, 1000), (1000, 8, 1000), (257, 200, 1030)]


def _check_linear(x, w, b, name, r, dy, bits=0):
    inner = w.size(1)
    dtype = x.dtype
    y, z = linear_forward(x, w, b, name, r, keep=True, bits=bits)
    X, W = x.double().reshape(-1, inner), w.double()
    Z = X @ W.t() + (0 if b is None else b.double())
    S = X.abs() @ W.abs().t() + (0 if b is None else b.double().abs())
    off = _c(inner, dtype) * S
    value = oracle.act(name, Z)
    # a slope is at most 1.13, erf and the like are good to a few units of 1 + |z|
    y_off = 1.13 * off + 16 * EPS32 * (1 + Z.abs())
    want = value if r is None else value + r.double().reshape(value.shape)
    _within(y.reshape(want.shape), want, y_off + 2 * EPS32 * want.abs() + (0 if r is None else 2 * EPS32 * r.double().abs().reshape(want.shape)), "y")
    if name != "none":
        if bits:
            zv = oracle.values8(z.q, z.e, torch.float64)
            q, e = oracle.keep8(Z)
            step = torch.exp2(torch.maximum(z.e.double(), e.double()) - 127).repeat_interleave(32, 1)[:, :Z.size(1)]
            assert torch.all((zv - Z).abs() <= step / 2 + off), "kept z"     # half a step, and what z itself is off
        else:
            zv = z.double()
            _within(z, Z, off, "z")
    else:
        zv = Z
    dx, dw, db = linear_backward(dy, x, w, name, z)
    G = dy.double().reshape(Z.shape)
    slope = oracle.act_slope(name, zv)
    dz = G * slope
    dz_off = (16 * EPS32 * G.abs() * (1 + zv.abs()) if name != "none" else 0 * G)
    rounded = dz_off + (U[dtype] * dz.abs() if name != "none" and dtype != torch.float32 else 0) + (LEAST[dtype] if name != "none" else 0)
    outer, rows = w.size(0), X.size(0)
    _within(dx.reshape(X.shape), dz @ W, (rounded @ W.abs()) * 1.01 + _c(outer, dtype) * (dz.abs() @ W.abs()), "dx")
    _within(dw, dz.t() @ X, (rounded.t() @ X.abs()) * 1.01 + _c(rows, dtype) * (dz.abs().t() @ X.abs()), "dw")
    _within(db, dz.sum(0), dz_off.sum(0) + 64 * EPS32 * dz.abs().sum(0), "db")
    assert status() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,inner,outer", SHAPES)
def test_linear(dtype, rows, inner, outer):
    i = SHAPES.index((rows, inner, outer))
    name = ["none", "gelu", "relu", "silu", "gelu_tanh"][i % 5]
    _check_linear(_randn(rows, inner, dtype=dtype), _randn(outer, inner, dtype=dtype, scale=inner ** -0.5, seed=1),
                  _randn(outer, dtype=dtype, seed=2) if i % 3 else None, name, _randn(rows, outer, dtype=dtype, seed=3) if i % 2 else None,
                  _randn(rows, outer, dtype=dtype, seed=4), bits=8 * (i % 4 > 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("bits", [0, 8])
def test_linear_activations(dtype, name, bits):
    x, w = _randn(70, 96, dtype=dtype), _randn(100, 96, dtype=dtype, scale=0.2, seed=1)
    _check_linear(x, w, _randn(100, dtype=dtype, seed=2), name, _randn(70, 100, dtype=dtype, seed=3), _randn(70, 100, dtype=dtype, seed=4), bits)


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_strides_and_addresses(dtype):
    """Rows apart, bases and rows off 16-byte boundaries, transposed weights, more axes."""
    x, w, dy = _randn(40, 200, dtype=dtype), _randn(72, 200, dtype=dtype, scale=0.1, seed=1), _randn(40, 200, dtype=dtype, seed=2)
    _check_linear(x[:, 8:72], w[:, 64:128], None, "gelu", None, dy[:, :72])
    _check_linear(x[:, 3:67], w[:, 1:65], None, "gelu", dy[:, 100:172], dy[:, 5:77])
    _check_linear(x[::2, ::2], w[:, ::2], w[:, 3], "silu", None, dy[::2, 1:73])
    _check_linear(x[:, :72], w.t()[:100, :], None, "relu", None, dy[:, :100])
    _check_linear(_randn(3, 4, 64, dtype=dtype).transpose(0, 1), w[:, :64], None, "none", None, _randn(3, 4, 72, dtype=dtype).transpose(0, 1))
    _check_linear(_randn(1, 64, dtype=dtype).expand(9, 64), w[:, :64], None, "none", None, _randn(1, 72, dtype=dtype).expand(9, 72))
    _check_linear(_randn(64, dtype=dtype), w[:, :64], None, "gelu", None, _randn(72, dtype=dtype))


def test_linear_f32_keeps_f32s_accuracy():
    """K = 10000, operands of the extremes of f32's range: three pieces carry 24 bits at any scale."""
    x, w = _randn(40, 10000), _randn(50, 10000, seed=1)
    y, _ = linear_forward(x, w)
    want = x.double() @ w.double().t()
    assert float((y - want).norm() / want.norm()) < 1e-6
    scale = torch.tensor([1e30, 1e-30, 1.0, 3e37] * 10, device=DEV)[:, None]
    y, _ = linear_forward(x * scale, w * 1e-3)
    want = (x * scale).double() @ (w * 1e-3).double().t()
    rel = (y.double() - want).norm(dim=1) / want.norm(dim=1)
    assert float(rel[[i for i in range(40) if i % 4 != 1]].max()) < 1e-6
    assert float(rel.max()) < 1e-5      # at 1e-33 the last piece of x reaches the end of bf16's range, 2^-133
    big = torch.full((1, 32), torch.finfo(torch.float32).max, device=DEV)
    assert torch.equal(linear_forward(big, torch.eye(32, device=DEV))[0], big)     # rounding its first piece would overflow


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_not_finite_stays_in_its_row(dtype):
    x, w = _randn(200, 96, dtype=dtype), _randn(64, 96, dtype=dtype, seed=1)
    x[5, 3], x[150, 90] = math.inf, math.nan
    y, _ = linear_forward(x, w)
    good = [i for i in range(200) if i not in (5, 150)]
    assert not torch.isfinite(y[5]).any() and torch.isnan(y[150]).all()
    assert torch.isfinite(y[good]).all() and torch.equal(y[good], linear_forward(torch.nan_to_num(x, 0, 0, 0), w)[0][good])
    _, z = linear_forward(x, w, None, "gelu", keep=True, bits=8)
    assert z.restore()[150].isnan().all() and z.restore()[good].isfinite().all()
    # rows past the end are not read as anything but zero: the same product in a larger buffer of NaN
    for rows in (3, 100):
        room = torch.full((400, 96), math.nan, device=DEV, dtype=dtype)
        room[:rows] = x[10:10 + rows]
        assert torch.equal(linear_forward(room[:rows], w)[0], linear_forward(x[10:10 + rows].clone(), w)[0])
    room = torch.full((200, 104), math.nan, device=DEV, dtype=dtype)
    room[:, :96] = torch.nan_to_num(x, 0, 0, 0)
    assert torch.equal(linear_forward(room[:, :96], w)[0][good], y[good])


@pytest.mark.parametrize("rows,inner,outer", [(40, 1500, 600), (512, 1024, 1024), (1100, 1500, 1400)])
def test_linear_f32_entries_of_unequal_size(rows, inner, outer):
    """One entry of a row may be as large as f32 holds without a loss to the others, where its partner is zero: a masked
    token's values, an unused channel.  Every entry of a result is held to the sum of its own products' magnitudes."""
    x, w, dy = _randn(rows, inner), _randn(outer, inner, scale=inner ** -0.5, seed=1), _randn(rows, outer, seed=2)
    x[:, 7] = 2.0 ** 30                 # a channel of x that no weight reads
    w[:, 7] = 0
    w[5] *= 2.0 ** 20                   # an output that no gradient reaches
    dy[:, 5] = 0
    x[3] = 2.0 ** 60                    # a token that no gradient reaches
    dy[3] = 0
    X, W, D = x.double(), w.double(), dy.double()
    y = linear_forward(x, w)[0]
    dx, dw, _ = linear_backward(dy, x, w)
    _within(y, X @ W.t(), _c(inner, x.dtype) * (X.abs() @ W.abs().t()), "y")
    _within(dx, D @ W, _c(outer, x.dtype) * (D.abs() @ W.abs()), "dx")
    _within(dw, D.t() @ X, _c(rows, x.dtype) * (D.abs().t() @ X.abs()), "dw")


def _infinite(got, want, what):
    assert torch.equal(got.isnan().cpu(), want.isnan().cpu()), what + ": NaN"
    assert torch.equal(torch.where(got.isinf(), got, 0).double().cpu(), torch.where(want.isinf(), want, 0).cpu()), what + ": infinities"


def _with_infinities(rows, cols, seed):
    """Infinities, zeros opposite them, values with one, two and three pieces, of both signs and unequal size."""
    m = _randn(rows, cols, seed=seed) * torch.exp(3 * _randn(rows, cols, seed=seed + 1))
    gen = torch.Generator(device=DEV).manual_seed(seed)
    pick = torch.rand(rows, cols, device=DEV, generator=gen)
    m = torch.where(pick < 0.2, m.round(), torch.where(pick < 0.4, m.bfloat16().float(), m))
    where = torch.rand(rows, cols, device=DEV, generator=gen)
    m[where < 0.5 / cols] = math.inf
    m[(where >= 0.5 / cols) & (where < 1 / cols)] = -math.inf
    return m


def _check_infinities(rows, inner, outer):
    x, w, dy = _with_infinities(rows, inner, 1), _with_infinities(outer, inner, 3), _with_infinities(rows, outer, 5)
    x[0, 0], w[0, 0], w[0, 1:], dy[0, 0] = math.inf, 1.0, 0.0, -math.inf
    X, W, D = x.double(), w.double(), dy.double()
    y = linear_forward(x, w)[0]
    _infinite(y, X @ W.t(), "y")
    assert y.isinf().any()
    dx, dw, _ = linear_backward(dy, x, w)
    _infinite(dx, D @ W, "dx")
    _infinite(dw, D.t() @ X, "dw")


@pytest.mark.parametrize("rows,inner,outer", [(1, 40, 33), (8, 64, 100), (20, 301, 130), (32, 128, 64), (70, 96, 130), (300, 700, 257)])
def test_linear_f32_infinities(rows, inner, outer):
    """An infinity times what is not zero is an infinity of its sign, though operands are multiplied in pieces."""
    _check_infinities(rows, inner, outer)


@pytest.mark.parametrize("rows,inner,outer", [(70, 96, 130), (300, 700, 257)])
def test_linear_f32_infinities_by_pairs(rows, inner, outer, monkeypatch):
    from gtopkssgd_b200.ops import linear as module
    monkeypatch.setattr(module, "PAIRS_FROM_FORWARD", 0)
    monkeypatch.setattr(module, "PAIRS_FROM_BACKWARD", 0)
    _check_infinities(rows, inner, outer)


@pytest.mark.parametrize("by_pairs", [False, True])
@pytest.mark.parametrize("rows", [5, 70])
def test_linear_f32_products_past_the_range(rows, by_pairs, monkeypatch):
    """An infinity of its sign, as of the sum in f32, whatever the lower pieces' signs."""
    from gtopkssgd_b200.ops import linear as module
    if by_pairs:
        monkeypatch.setattr(module, "PAIRS_FROM_FORWARD", 0)
    x, w = _randn(rows, 64).abs() + 0.1, _randn(40, 64, seed=1).abs() + 0.1
    sign = torch.where(torch.arange(40, device=DEV) % 2 == 0, 1.0, -1.0)[:, None]
    y = linear_forward(x * 1e25, w * sign * 1e25)[0]
    assert torch.equal(y, torch.full_like(y, math.inf) * sign.t())
    y = linear_forward(x * 1e15, w * sign * 1e15)[0]
    assert y.isfinite().all() and torch.equal(y.sign(), sign.t().expand_as(y))


@pytest.mark.parametrize("rows,inner,outer", [(1, 40, 33), (20, 1500, 600), (129, 65, 257), (515, 1001, 130), (1000, 8, 1000), (300, 2000, 96)])
def test_linear_f32_by_pairs(rows, inner, outer, monkeypatch):
    """f32 operands as two scaled f16 pieces, which only large products take, at the sizes where they can go wrong.  What
    the three products leave out is 2^-24 of a product's magnitude at most, and the pieces are off by as much."""
    from gtopkssgd_b200.ops import linear as module
    monkeypatch.setattr(module, "PAIRS_FROM_FORWARD", 0)
    monkeypatch.setattr(module, "PAIRS_FROM_BACKWARD", 0)
    for scale in (1.0, 1e30, 1e-30):
        x, w = _randn(rows, inner, scale=scale), _randn(outer, inner, scale=inner ** -0.5 / scale, seed=1)
        x *= torch.exp(4 * _randn(rows, 1, seed=8))                 # rows of unequal size
        dy = _randn(rows, outer, seed=2) * torch.exp(4 * _randn(1, outer, seed=9))
        _check_linear(x, w, _randn(outer, seed=3), "none", _randn(rows, outer, seed=4), dy)
        _check_linear(x, w, None, "gelu", None, dy, 8)
    x[0, 0], dy[-1, -1] = math.inf, math.nan
    y = linear_forward(x, w)[0]
    dx, dw, _ = linear_backward(dy, x, w)
    assert not torch.isfinite(y[0]).any() and torch.isfinite(y[1:]).all()
    assert torch.isnan(dx[-1]).all() and torch.isfinite(dx[:-1]).all() and torch.isnan(dw[-1]).all()
    x = _randn(rows, inner)
    got, want = linear_backward(dy[:, :outer].nan_to_num(), Activation8.keep(x), w)[1], linear_backward(dy.nan_to_num(), Activation8.keep(x).restore(), w)[1]
    assert torch.equal(got, want)


def test_linear_f32_by_pairs_keeps_f32s_accuracy(monkeypatch):
    from gtopkssgd_b200.ops import linear as module
    monkeypatch.setattr(module, "PAIRS_FROM_FORWARD", 0)
    monkeypatch.setattr(module, "PAIRS_FROM_BACKWARD", 0)
    x, w = _randn(40, 10000), _randn(50, 10000, seed=1)
    for scale in (1.0, 1e30, 1e-30):
        y = linear_forward(x * scale, w / scale)[0]
        want = (x * scale).double() @ (w / scale).double().t()
        assert float((y - want).norm() / want.norm()) < 1e-6
    big = torch.full((1, 32), torch.finfo(torch.float32).max, device=DEV)
    assert torch.equal(linear_forward(big, torch.eye(32, device=DEV))[0], big)
    zeros = torch.zeros(3, 32, device=DEV)
    assert torch.equal(linear_forward(zeros, torch.eye(32, device=DEV))[0], zeros)


@pytest.mark.parametrize("bits", [0, 8])
def test_feed_forward_block_by_pairs(bits, monkeypatch):
    from gtopkssgd_b200.ops import linear as module
    monkeypatch.setattr(module, "PAIRS_FROM_FORWARD", 0)
    monkeypatch.setattr(module, "PAIRS_FROM_BACKWARD", 0)
    for rows, dim, hidden in ((1, 40, 33), (70, 101, 203), (300, 64, 256)):
        test_feed_forward_block(torch.float32, bits, rows, dim, hidden)


def test_linear_needs_and_8_bit_input():
    x, w, dy = _randn(60, 100), _randn(40, 100, seed=1), _randn(60, 40, seed=2)
    z = linear_forward(x, w, None, "gelu", keep=True)[1]
    full = linear_backward(dy, x, w, "gelu", z)
    for i in range(8):
        need = (bool(i & 1), bool(i & 2), bool(i & 4))
        got = linear_backward(dy, x, w, "gelu", z, need)
        for n, a, b in zip(need, got, full):
            assert (a is None and not n) or torch.equal(a, b)
    kept = Activation8.keep(x)
    got, want = linear_backward(dy, kept, w, "gelu", z)[1], linear_backward(dy, kept.restore(), w, "gelu", z)[1]
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)     # the same numbers, as one piece and as three
    empty = torch.empty(0, 100, device=DEV)
    assert linear_forward(empty, w)[0].shape == (0, 40)
    dx, dw, db = linear_backward(torch.empty(0, 40, device=DEV), empty, w)
    assert dx.shape == (0, 100) and not dw.any() and not db.any()


# -- block ------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bits", [0, 8])
@pytest.mark.parametrize("rows,dim,hidden", [(1, 40, 33), (35, 300, 1200), (70, 101, 203), (300, 64, 256), (400, 1500, 40), (5, 9000, 24), (3, 16400, 16)])
def test_feed_forward_block(dtype, bits, rows, dim, hidden):
    """Against the formulas in 64 bits at the kept values.  Five roundings to the type lie between dy and a gradient
    (dz, the hidden layer or the norm's output, da, and the result's own), each of relative size u; in the 2-norm of
    a whole gradient they add up to 5 u at most.  f32: sums of up to 1200 terms, 1e-6."""
    x = _randn(rows, dim, dtype=dtype)
    p = [_randn(dim, dtype=dtype, seed=1) * 0.1 + 1, _randn(dim, dtype=dtype, seed=2) * 0.1, _randn(hidden, dim, dtype=dtype, scale=dim ** -0.5, seed=3),
         _randn(hidden, dtype=dtype, seed=4) * 0.1, _randn(dim, hidden, dtype=dtype, scale=hidden ** -0.5, seed=5), _randn(dim, dtype=dtype, seed=6) * 0.1]
    dy = _randn(rows, dim, dtype=dtype, seed=7)
    y, kept = feed_forward(x, *p, activation="gelu", bits=bits)
    got = feed_forward_backward(dy, kept, *p[:3], p[4], "gelu")
    g, b, w1, b1, w2, b2 = (t.double() for t in p)
    want_y = x.double() + F.linear(F.gelu(F.linear(F.layer_norm(x.double(), (dim,), g, b, 1e-5), w1, b1)), w2, b2)
    limit = max(1e-6, 5 * U[dtype])

    def near(a, e, what):
        assert a.dtype == dtype and a.shape == e.shape
        assert float((a.double() - e).norm()) <= limit * float(e.norm()), what

    near(y, want_y, "y")
    X, z = (oracle.values8(t.q, t.e, torch.float64) if bits else t.double() for t in (kept.x, kept.z))
    m, r, D = kept.mean.double()[:, None], kept.rstd.double()[:, None], dy.double()
    dz = (D @ w2) * oracle.act_slope("gelu", z)
    xh = (X - m) * r
    da = dz @ w1
    t = da * g
    dx = r * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True)) + D
    for a, e, what in zip(got, (dx, (da * xh).sum(0), da.sum(0), dz.t() @ (xh * g + b), dz.sum(0), D.t() @ F.gelu(z), D.sum(0)),
                          ("dx", "dg", "db", "dw1", "db1", "dw2", "db2")):
        near(a, e, what)
    leaves = [v.clone().requires_grad_() for v in (x, *p)]
    out = feed_forward_block(*leaves, "gelu", 1e-5, bits)
    out.backward(dy)
    assert torch.equal(out, y) and all(torch.equal(v.grad, a) for v, a in zip(leaves, got))


@pytest.mark.parametrize("dtype,bits,by_pairs", [(torch.float32, 0, False), (torch.float32, 8, True), (torch.bfloat16, 8, False)])
@pytest.mark.parametrize("rows,dim,hidden", [(70, 101, 203), (130, 64, 96), (3, 16400, 16)])
def test_feed_forward_block_needs(dtype, bits, by_pairs, rows, dim, hidden, monkeypatch):
    """Any set of gradients is what it is among all of them (sums over rows and the norm's output may be made another way: two
    roundings of the type), and what nobody wants costs no product."""
    from gtopkssgd_b200.ops import lib
    from gtopkssgd_b200.ops import linear as module
    if by_pairs:
        monkeypatch.setattr(module, "PAIRS_FROM_BACKWARD", 0)
    x, dy = _randn(rows, dim, dtype=dtype), _randn(rows, dim, dtype=dtype, seed=7)
    p = [_randn(dim, dtype=dtype, seed=1), _randn(dim, dtype=dtype, seed=2), _randn(hidden, dim, dtype=dtype, scale=dim ** -0.5, seed=3),
         _randn(hidden, dtype=dtype, seed=4), _randn(dim, hidden, dtype=dtype, scale=hidden ** -0.5, seed=5), _randn(dim, dtype=dtype, seed=6)]
    kept = feed_forward(x, *p, bits=bits)[1]
    full = feed_forward_backward(dy, kept, *p[:3], p[4])
    limit = max(1e-6, 4 * U[dtype])
    for i in range(128):
        need = tuple(bool(i >> j & 1) for j in range(7))
        for n, a, b in zip(need, feed_forward_backward(dy, kept, *p[:3], p[4], need=need), full):
            assert (a is None) != n and (a is None or float((a.double() - b.double()).norm()) <= limit * float(b.double().norm())), need

    def products(*trained):
        leaves = [v.clone().requires_grad_(i in trained) for i, v in enumerate((x, *p))]
        y = feed_forward_block(*leaves, "gelu", 1e-5, bits)
        calls = []
        run = lib.calls()
        with monkeypatch.context() as patch:
            patch.setattr(lib, "calls", lambda: type("Calls", (), {"__getattr__": lambda self, name: calls.append(name) or getattr(run, name)})())
            y.backward(dy)
        assert all((v.grad is not None) == (i in trained) for i, v in enumerate(leaves))
        return calls.count("gtk_k8_gemm")

    assert products(*range(7)) == 4 and products(0, 1, 2) == 2 and products(0) == 2 and products(3) == 2 and products(5) == 2 and products(4) == 1
    assert products(6) == 0


def test_gradients_against_differences():
    """Central differences of the 64-bit function along a direction, against the f32 kernels' gradients."""
    rows, dim, hidden = 12, 48, 96
    args = [_randn(rows, dim), _randn(dim, seed=1), _randn(dim, seed=2), _randn(hidden, dim, scale=0.2, seed=3), _randn(hidden, seed=4),
            _randn(dim, hidden, scale=0.2, seed=5), _randn(dim, seed=6)]
    dy = _randn(rows, dim, seed=7).double()

    def f(x, g, b, w1, b1, w2, b2):
        return (dy * (x + F.linear(F.gelu(F.linear(F.layer_norm(x, (dim,), g, b, 1e-5), w1, b1)), w2, b2))).sum()

    leaves = [v.clone().requires_grad_() for v in args]
    feed_forward_block(*leaves).backward(dy.float())
    h = 1e-5
    for i, leaf in enumerate(leaves):
        d = _randn(*leaf.shape, seed=20 + i).double()
        moved = [[v.double() + (s * h * d if j == i else 0) for j, v in enumerate(args)] for s in (1, -1)]
        slope = float((f(*moved[0]) - f(*moved[1])) / (2 * h))
        size = float((leaf.grad.double().abs() * d.abs()).sum())
        assert abs(float((leaf.grad.double() * d).sum()) - slope) <= 1e-5 * size, i   # differences: h^2; gradient: f32 sums


# -- use --------------------------------------------------------------------------------
def test_streams_graphs_and_repetition():
    """On another stream, captured and replayed on new inputs, and twice the same bits."""
    x = _randn(300, 200).requires_grad_()
    p = [_randn(200, seed=1), _randn(200, seed=2), _randn(333, 200, seed=3), _randn(333, seed=4), _randn(200, 333, seed=5), _randn(200, seed=6)]

    def step(inp):
        return feed_forward_backward(inp, feed_forward(inp, *p, bits=8)[1], p[0], p[1], p[2], p[4])

    with torch.no_grad():
        want = step(x)
        assert all(torch.equal(a, b) for a, b in zip(step(x), want))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(x)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        static = torch.zeros_like(x)
        graph = torch.cuda.CUDAGraph()
        step(static)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = step(static)
        static.copy_(x)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        torch.cuda.synchronize()
    assert status() == 0


def test_what_is_kept_in_8_bits_is_let_go():
    """The copies, 33 bytes for 32 columns or what is left of them, are held until the backward pass and no longer, though the
    result is; hooks may move them, and what comes back without the rows' padding is read as well."""
    def held():
        return torch.cuda.memory_stats()["requested_bytes.all.current"]

    rows, hidden = 300, 200
    for width in (1500, 101):
        x, p = _randn(rows, width), [_randn(width, seed=1), _randn(width, seed=2), _randn(hidden, width, scale=width ** -0.5, seed=3), _randn(hidden, seed=4),
                                     _randn(width, hidden, scale=hidden ** -0.5, seed=5), _randn(width, seed=6)]
        leaves = [v.requires_grad_() for v in (x, *p)]
        copies = sum(33 * rows * -(-n // 32) for n in (width, hidden))
        for run, more in ((lambda: linear(x, p[2], p[3], "gelu", bits=8), 0), (lambda: feed_forward_block(x, *p, "gelu", 1e-5, 8), 8 * rows)):
            for v in leaves:
                v.grad = None
            run().sum().backward()
            want = [None if v.grad is None else v.grad.clone() for v in leaves]
            before = held()
            y = run()
            assert held() - before == y.untyped_storage().nbytes() + copies + more
            y.sum().backward()      # into gradients that are there
            assert held() - before == y.untyped_storage().nbytes()
            for v in leaves:
                v.grad = None
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().contiguous(), lambda t: t.to(DEV)):
                run().sum().backward()
            for v, g in zip(leaves, want):
                assert (v.grad is None) == (g is None) and (g is None or torch.allclose(v.grad, g, rtol=1e-5, atol=1e-5 * float(g.abs().max())))
            del y


def test_matrices_over_2_31_elements():
    """Offsets past 32 bits: the last rows of 8-bit copies, norms and products."""
    rows, cols = 70001, 32768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-2:] = _randn(2, cols, dtype=torch.bfloat16)
    kept = Activation8.keep(x)
    want = oracle.restore8(*oracle.keep8(x[-2:]), torch.bfloat16)
    assert torch.equal(kept.restore()[-2:], want) and not kept.q[:-2:1000].any()
    del kept
    x = x.view(-1, 1024)
    y = layer_norm_forward(x)[0]
    assert torch.equal(y[-64:], layer_norm_forward(x[-64:])[0]) and not y[:-64:1000].any()
    del y
    w = _randn(40, 1024, dtype=torch.bfloat16, seed=1)
    y = linear_forward(x, w)[0]
    X, W = x[-64:].double(), w.double()
    _within(y[-64:], X @ W.t(), _c(1024, x.dtype) * (X.abs() @ W.abs().t()), "y")
    del x, y
    a, w = _randn(rows, 8, dtype=torch.bfloat16), _randn(32768, 8, dtype=torch.bfloat16, seed=1)
    y = linear_forward(a, w)[0]
    assert torch.equal(y[-64:], linear_forward(a[-64:], w)[0])
    dx, dw, _ = linear_backward(y, a, w)
    Y, W = y[-64:].double(), w.double()
    _within(dx[-64:], Y @ W, _c(32768, dx.dtype) * (Y.abs() @ W.abs()), "dx")   # k is split differently over more rows
    want = y[:, -64:].double().t() @ a.double()
    assert float((dw[-64:] - want).norm() / want.norm()) < 1e-2


def test_empty_axes_on_the_gpu():
    from test_layers_cpu import _check_empty
    _check_empty(DEV)


def test_products_of_no_known_form_are_refused():
    """By the host, before anything is launched: f32 results have pieces, pairs their scales, and both operands fit."""
    from gtopkssgd_b200.ops import lib
    a, out = torch.zeros(64, 64, dtype=torch.bfloat16, device=DEV), torch.full((64, 64), 7.0, device=DEV)

    def call(code, half, pieces, n=64, ld=64):
        at = a.data_ptr()
        return lib.calls().gtk_k8_gemm(code, half, 64, n, 64, at, ld, pieces[0], 0, 0, None, at, ld, pieces[1], 0, 0, None, out.data_ptr(), 64, None, None, 0,
                                       0, 0, None, 0, None, 0, None, 0, None, 0, None, None, 10 ** 9, torch.cuda.current_stream().cuda_stream)

    for args in ((0, 0, (1, 1)), (0, 1, (1, 1)), (0, 1, (2, 2)), (0, 0, (1, 3)), (0, 0, (3, 3)), (2, 0, (3, 1)), (0, 1, (2, 1)), (2, 0, (1, 1), 0), (2, 0, (1, 1), 64, 60)):
        assert call(*args) == -1, args
    assert bool((out == 7).all()) and status() == 0


def test_refusals_on_the_gpu():
    x, w = _randn(8, 64), _randn(16, 64)
    with pytest.raises(TypeError):
        layer_norm(x.double())
    with pytest.raises(TypeError):
        Activation8.keep(x.long())
    with pytest.raises(ValueError):
        linear(x, w.cpu())
    with pytest.raises(ValueError):
        layer_norm(x, torch.ones(64))
    with pytest.raises(ValueError):
        linear(x, w.half())
    _, mean, rstd = layer_norm_forward(x)
    with pytest.raises(TypeError):
        layer_norm_backward(x, x, mean.double(), rstd)


def test_language_model_with_blocks_in_a_sparse_training_step(monkeypatch):
    """The PTB model with a block behind the LSTM, gTop-k: the losses follow those with the block in library functions
    (f32: to 1e-3 over ten steps; 8 bits, and bf16 inside: to 2e-2), and fall."""
    from gtopkssgd_b200.models import feed_forward as module
    from gtopkssgd_b200.models import lstm
    from gtopkssgd_b200.parallel.compression import compressors
    from gtopkssgd_b200.parallel.distributed_optimizer import DistributedOptimizer

    def library(x, g, b, w1, b1, w2, b2, activation, eps, bits):
        return x + F.linear(F.gelu(F.linear(F.layer_norm(x, (x.size(-1),), g, b, eps), w1, b1)), w2, b2)

    def losses(bits, dtype):
        torch.manual_seed(0)
        net = lstm(vocab_size=50, embedding_dim=100, num_steps=5, batch_size=4, ff_layers=1, ff_dim=400, ff_bits=bits, ff_dtype=dtype).to(DEV)
        opt = DistributedOptimizer(torch.optim.SGD(net.parameters(), lr=0.05), net.named_parameters(), compression=compressors["gtopk"], is_sparse=True,
                                   density=0.05)
        tokens = torch.randint(0, 50, (6, 4), device=DEV)
        got = []
        for _ in range(60):
            opt.zero_grad()
            logits, _ = net(tokens[:-1], net.init_hidden())
            loss = F.cross_entropy(logits.view(-1, 50), tokens[1:].reshape(-1))
            loss.backward()
            opt.step()
            got.append(float(loss.detach()))
        opt.check_status()
        opt.stop()
        return got

    cases = ((0, None, 1e-3), (8, None, 2e-2), (8, torch.bfloat16, 2e-2))
    got = [losses(bits, dtype) for bits, dtype, _ in cases]
    assert status() == 0
    monkeypatch.setattr(module, "feed_forward_block", library)
    want = losses(0, None)
    for g, (_, _, off) in zip(got, cases):
        assert all(abs(a - b) <= off * b for a, b in zip(g[:10], want)) and g[-1] < 0.97 * g[0]


# -- what runs out ------------------------------------------------------------------------
def test_a_wait_that_runs_out_is_told_to_the_whole_warp():
    """Lanes of an epilogue's warp that go on while others give up would wait for them without end: one answer for all."""
    from gtopkssgd_b200.ops.linear import clear_status, rehearse_timeout
    assert status() == 0
    answers = rehearse_timeout(DEV, limit_ms=5)
    assert answers.tolist() == [0] * 32 and status() == 6
    clear_status()
    x, w = _randn(70, 64), _randn(40, 64, seed=1)
    y = linear_forward(x, w)[0]
    _within(y, x.double() @ w.double().t(), _c(64, x.dtype) * (x.double().abs() @ w.double().abs().t()), "y")
    assert status() == 0


def test_a_wait_that_runs_out_reaches_the_optimizer():
    from gtopkssgd_b200.ops.lib import GtopkNativeError
    from gtopkssgd_b200.ops.linear import check_status, clear_status, rehearse_timeout
    from gtopkssgd_b200.parallel.compression import compressors
    from gtopkssgd_b200.parallel.distributed_optimizer import DistributedOptimizer
    net = torch.nn.Linear(8, 4).to(DEV)
    opt = DistributedOptimizer(torch.optim.SGD(net.parameters(), lr=0.1), net.named_parameters(), compression=compressors["gtopk"], is_sparse=True,
                               density=0.1)
    opt.check_status()
    rehearse_timeout(DEV, limit_ms=5)
    for check in (opt.check_status, check_status):
        with pytest.raises(GtopkNativeError):
            check()
    clear_status()
    opt.check_status()
    opt.stop()
