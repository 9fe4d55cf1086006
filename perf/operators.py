"""The operators of a feed-forward block in training, as timed cases.

Four kinds of pass, each through the public entry points:

``norm``    layer norm over the last axis: ``layer_norm_forward`` and, for a
            training step, ``layer_norm_backward`` with the gradients of weight
            and bias.
``linear``  act(x W^T + bias) + residual: ``linear_forward`` and, for a training
            step, ``linear_backward``, which reads what the forward pass kept of
            the activation's input (in the inputs' type, or in 8 bits).
``keep``    an activation kept in 8 bits: ``Activation8.keep``, ``restore``, and
            the gradient through the activation and the bias that were before it
            (``Activation8.backward``).
``block``   y = x + W2 act(W1 norm(x) + b1) + b2: ``feed_forward`` with what it
            keeps for the backward pass, or ``feed_forward_backward`` from what a
            forward pass had kept.

The 8-bit form: blocks of 32 along a row share a power of two 2^e, the least with
max|x| <= 127 * 2^e; a value is rint(x / 2^e) * 2^e.
"""
from __future__ import annotations

import math
import random

import torch
import torch.nn.functional as F

own = False

DEV = "cuda"
BLOCK = 32
EPS = 1e-5
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one step of the PTB language model's 20 sequences, hidden size 1500: the smallest call, latency
        {"name": "norm-20x1500-f32-forward", "op": "norm", "rows": 20, "cols": 1500, "type": "f32", "train": False},
        # the PTB batch, 35 steps of 20 sequences, in the framework's own type
        {"name": "norm-700x1500-f32", "op": "norm", "rows": 700, "cols": 1500, "type": "f32", "train": True},
        # odd sizes: rows that begin at no wide boundary
        {"name": "norm-1237x1021-f16", "op": "norm", "rows": 1237, "cols": 1021, "type": "f16", "train": True},
        # a large batch, far more than the second-level cache holds
        {"name": "norm-16384x4096-bf16", "op": "norm", "rows": 16384, "cols": 4096, "type": "bf16", "train": True},
        # 20 rows through a first feed-forward layer: the weights' bytes and latency count
        {"name": "linear-20x1500x6000-bf16-forward", "op": "linear", "rows": 20, "inner": 1500, "outer": 6000, "type": "bf16",
         "act": "relu", "residual": False, "bits": 0, "train": False},
        # the PTB model's softmax layer: 10 000 words, no activation, f32 as the framework trains it
        {"name": "linear-700x1500x10000-f32", "op": "linear", "rows": 700, "inner": 1500, "outer": 10000, "type": "f32",
         "act": "none", "residual": False, "bits": 0, "train": True},
        # odd sizes in every direction, with a residual
        {"name": "linear-515x1001x2047-f16", "op": "linear", "rows": 515, "inner": 1001, "outer": 2047, "type": "f16",
         "act": "silu", "residual": True, "bits": 0, "train": True},
        # a large layer whose pre-activation is kept in 8 bits
        {"name": "linear-8192x2048x8192-bf16-8bit", "op": "linear", "rows": 8192, "inner": 2048, "outer": 8192, "type": "bf16",
         "act": "gelu", "residual": False, "bits": 8, "train": True},
        # 8-bit copy of the PTB batch's hidden layer
        {"name": "keep-700x6000-f32", "op": "keep", "rows": 700, "cols": 6000, "type": "f32", "act": "gelu"},
        # the same of a large batch
        {"name": "keep-16384x8192-bf16", "op": "keep", "rows": 16384, "cols": 8192, "type": "bf16", "act": "gelu"},
        # the whole block, PTB batch, forward pass with its 8-bit checkpoints
        {"name": "block-700x1500x6000-bf16-forward", "op": "block", "rows": 700, "inner": 1500, "outer": 6000, "type": "bf16",
         "act": "gelu", "bits": 8, "backward": False},
        # its backward pass from the checkpoints, large
        {"name": "block-8192x2048x8192-bf16-backward", "op": "block", "rows": 8192, "inner": 2048, "outer": 8192, "type": "bf16",
         "act": "gelu", "bits": 8, "backward": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["norm", "linear", "linear", "keep", "block", "block"])
    kind = rng.choice(["f32", "bf16", "f16"])
    act = rng.choice(["relu", "gelu", "gelu_tanh", "silu"])
    if op in ("norm", "keep"):
        cols = _log_int(rng, 33, 12000)
        rows = _log_int(rng, 1, max(2, min(16384, 100_000_000 // (cols * 4))))
        if op == "norm":
            return {"op": op, "rows": rows, "cols": cols, "type": kind, "train": rng.random() < 0.7}
        return {"op": op, "rows": rows, "cols": cols, "type": kind, "act": act}
    while True:
        rows, inner, outer = _log_int(rng, 1, 8192), _log_int(rng, 40, 4096), _log_int(rng, 40, 10000)
        if rows * inner * outer <= 8192 * 2048 * 4096:
            break
    if rng.random() < 0.6:   # models' widths are as a rule multiples of 8; the others are odd as they come
        inner, outer = -(-inner // 8) * 8, -(-outer // 8) * 8
    if op == "linear":
        # codes of 8 bits stand for values that were computed in f32: where results are f32 too, the last bit of one value
        # would decide a whole step of its code, so the f32 cases keep the value
        return {"op": op, "rows": rows, "inner": inner, "outer": outer, "type": kind, "act": rng.choice(["none", act]),
                "residual": rng.random() < 0.5, "bits": 0 if kind == "f32" else rng.choice([0, 8]), "train": rng.random() < 0.7}
    backward = rng.random() < 0.6
    bits = rng.choice([0, 8]) if backward or kind != "f32" else 0
    return {"op": op, "rows": rows, "inner": inner, "outer": outer, "type": kind, "act": act, "bits": bits, "backward": backward}


# -- inputs -------------------------------------------------------------------
def _codes(x):
    """x in 8 bits: (codes, int8, rows by columns; exponents + 127, uint8, rows by blocks)."""
    rows, cols = x.shape
    padded = F.pad(x.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    mantissa, exponent = torch.frexp(padded.abs().amax(2))        # max = mantissa * 2^exponent, mantissa in [1/2, 1)
    e = torch.where(mantissa > 127 / 128, exponent - 6, exponent - 7)
    e = torch.where(mantissa == 0, torch.full_like(e, -127), e).clamp(min=-127)
    q = torch.round(torch.ldexp(padded, -e.unsqueeze(2))).to(torch.int8)
    return q.view(rows, -1)[:, :cols].contiguous(), (e + 127).to(torch.uint8)


def _values(q, e):
    """What codes stand for, f32."""
    rows, cols = q.shape
    padded = F.pad(q.float(), (0, -cols % BLOCK)).view(rows, -1, BLOCK)
    return torch.ldexp(padded, e.int().unsqueeze(2) - 127).view(rows, -1)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)
    t = TYPES[case["type"]]

    def noise(*shape, scale=1.0, mean=0.0):
        return torch.randn(*shape, device=DEV, generator=gen).mul_(scale).add_(mean)

    def stream(rows, cols):
        """A residual stream: channels of unequal size and mean."""
        x = noise(rows, cols)
        return x.mul_(noise(cols).mul_(0.5).exp_()).add_(noise(cols, scale=0.3)).to(t)

    s = dict(case)
    rows = case["rows"]
    if case["op"] == "norm":
        cols = case["cols"]
        s.update(x=stream(rows, cols), w=noise(cols, scale=0.1, mean=1.0).to(t), b=noise(cols, scale=0.1).to(t),
                 dy=noise(rows, cols, scale=1e-2).to(t))
    elif case["op"] == "linear":
        inner, outer = case["inner"], case["outer"]
        s.update(x=noise(rows, inner).to(t), w=noise(outer, inner, scale=inner ** -0.5).to(t), b=noise(outer, scale=0.1).to(t),
                 r=noise(rows, outer).to(t) if case["residual"] else None, dy=noise(rows, outer, scale=1e-2).to(t))
    elif case["op"] == "keep":
        cols = case["cols"]
        s.update(x=stream(rows, cols), dy=noise(rows, cols, scale=1e-2).to(t))
    else:
        inner, outer = case["inner"], case["outer"]
        s.update(x=stream(rows, inner), g=noise(inner, scale=0.1, mean=1.0).to(t), b=noise(inner, scale=0.1).to(t),
                 w1=noise(outer, inner, scale=inner ** -0.5).to(t), b1=noise(outer, scale=0.1).to(t),
                 w2=noise(inner, outer, scale=outer ** -0.5).to(t), b2=noise(inner, scale=0.1).to(t))
        if case["backward"]:   # what a forward pass had kept
            x = s["x"].float()
            mean = x.mean(1)
            rstd = torch.rsqrt(x.var(1, unbiased=False) + EPS)
            z = F.linear(((x - mean[:, None]) * rstd[:, None]).mul_(s["g"].float()).add_(s["b"].float()).to(t),
                         s["w1"], s["b1"])
            s.update(mean=mean, rstd=rstd, dy=noise(rows, inner, scale=1e-2).to(t))
            if case["bits"]:
                s["xq"], s["xe"] = _codes(s.pop("x"))
                s["zq"], s["ze"] = _codes(z)
            else:
                s["z"] = z
    return s


# -- plain forms --------------------------------------------------------------
def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    return z / (1 + torch.exp(-z))


def _act_slope(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    sg = 1 / (1 + torch.exp(-z))
    return sg * (1 + z * (1 - sg))


def _norm(x, w, b):
    mean = x.mean(1)
    centred = x - mean[:, None]
    rstd = torch.rsqrt((centred * centred).mean(1) + EPS)
    return centred * rstd[:, None] * w + b, mean, rstd


def _norm_gradients(dy, x, mean, rstd, w):
    xh = (x - mean[:, None]) * rstd[:, None]
    t = dy * w
    dx = rstd[:, None] * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def _plain(s):
    t = TYPES[s["type"]]
    f = {k: v.float() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if s["op"] == "norm":
        y, mean, rstd = _norm(f["x"], f["w"], f["b"])
        out = {"y": y.to(t), "mean": mean, "rstd": rstd}
        if s["train"]:
            dx, dw, db = _norm_gradients(f["dy"], f["x"], mean, rstd, f["w"])
            out.update(dx=dx.to(t), dw=dw.to(t), db=db.to(t))
        return out
    if s["op"] == "linear":
        z = f["x"] @ f["w"].t() + f["b"]
        y = _act(s["act"], z)
        out = {"y": (y + f["r"] if "r" in f else y).to(t)}
        if s["train"]:
            if s["bits"]:
                z = _values(*_codes(z))
            dz = f["dy"] * _act_slope(s["act"], z)
            out.update(dx=(dz @ f["w"]).to(t), dw=(dz.t() @ f["x"]).to(t), db=dz.sum(0).to(t))
        return out
    if s["op"] == "keep":
        x = _values(*_codes(f["x"]))
        dz = f["dy"] * _act_slope(s["act"], x)
        return {"x": x.to(t), "dz": dz.to(t), "db": dz.sum(0).to(t)}
    if not s["backward"]:
        a, mean, rstd = _norm(f["x"], f["g"], f["b"])
        z = a @ f["w1"].t() + f["b1"]
        y = _act(s["act"], z) @ f["w2"].t() + f["b2"] + f["x"]
        if s["bits"]:
            return {"y": y.to(t), "mean": mean, "rstd": rstd, "x": _values(*_codes(f["x"])).to(t), "z": _values(*_codes(z)).to(t)}
        return {"y": y.to(t), "mean": mean, "rstd": rstd, "z": z.to(t)}
    x, z = (_values(s["xq"], s["xe"]), _values(s["zq"], s["ze"])) if s["bits"] else (f["x"], f["z"])
    dy, mean, rstd = f["dy"], f["mean"], f["rstd"]
    h = _act(s["act"], z)
    dz = (dy @ f["w2"]) * _act_slope(s["act"], z)
    a = (x - mean[:, None]) * rstd[:, None] * f["g"] + f["b"]
    dx, dg, db = _norm_gradients(dz @ f["w1"], x, mean, rstd, f["g"])
    return {"dx": (dx + dy).to(t), "dg": dg.to(t), "db": db.to(t), "dw1": (dz.t() @ a).to(t), "db1": dz.sum(0).to(t),
            "dw2": (dy.t() @ h).to(t), "db2": dy.sum(0).to(t)}


# -- the framework's operators ------------------------------------------------
def _framework(s):
    from gtopkssgd_b200.ops.activation8 import Activation8
    from gtopkssgd_b200.ops.feed_forward import FeedForwardKept, feed_forward, feed_forward_backward
    from gtopkssgd_b200.ops.layer_norm import layer_norm_backward, layer_norm_forward
    from gtopkssgd_b200.ops.linear import linear_backward, linear_forward
    if s["op"] == "norm":
        y, mean, rstd = layer_norm_forward(s["x"], s["w"], s["b"], EPS)
        out = {"y": y, "mean": mean, "rstd": rstd}
        if s["train"]:
            out["dx"], out["dw"], out["db"] = layer_norm_backward(s["dy"], s["x"], mean, rstd, s["w"])
        return out
    if s["op"] == "linear":
        y, z = linear_forward(s["x"], s["w"], s["b"], s["act"], s["r"], keep=s["train"], bits=s["bits"])
        out = {"y": y}
        if s["train"]:
            out["dx"], out["dw"], out["db"] = linear_backward(s["dy"], s["x"], s["w"], s["act"], z)
        return out
    if s["op"] == "keep":
        kept = Activation8.keep(s["x"])
        dz, db = kept.backward(s["dy"], s["act"])
        return {"x": kept.restore(), "dz": dz, "db": db}
    if not s["backward"]:
        y, kept = feed_forward(s["x"], s["g"], s["b"], s["w1"], s["b1"], s["w2"], s["b2"], s["act"], EPS, bits=s["bits"])
        out = {"y": y, "mean": kept.mean, "rstd": kept.rstd}
        if s["bits"]:
            out.update(x=kept.x.restore(), z=kept.z.restore())
        else:
            out["z"] = kept.z
        return out
    t = TYPES[s["type"]]
    if s["bits"]:
        x, z = Activation8(s["xq"], s["xe"], t), Activation8(s["zq"], s["ze"], t)
    else:
        x, z = s["x"], s["z"]
    got = feed_forward_backward(s["dy"], FeedForwardKept(x, s["mean"], s["rstd"], z), s["g"], s["b"], s["w1"], s["w2"], s["act"])
    return dict(zip(("dx", "dg", "db", "dw1", "db1", "dw2", "db2"), got))


def run(state):
    return _framework(state) if own else _plain(state)


# -- what a pass cannot do without ----------------------------------------------
def work(case):
    size = 4 if case["type"] == "f32" else 2
    rows = case["rows"]
    if case["op"] in ("norm", "keep"):
        cols = case["cols"]
        one = rows * cols
        if case["op"] == "keep":   # x, dy in; the value, dz, db out
            return {"bytes": (4 * one + cols) * size, "flops": 24 * one}
        if not case["train"]:
            return {"bytes": (2 * one + 2 * cols) * size + 8 * rows, "flops": 8 * one}
        return {"bytes": (4 * one + 4 * cols) * size + 8 * rows, "flops": 22 * one}
    inner, outer = case["inner"], case["outer"]
    product = 2 * rows * inner * outer
    if case["op"] == "linear":
        values = rows * inner + inner * outer + outer + rows * outer * (2 if case["residual"] else 1)
        if not case["train"]:
            return {"bytes": values * size, "flops": product}
        return {"bytes": (values + rows * outer + rows * inner + inner * outer + outer) * size, "flops": 3 * product}
    weights = 2 * inner * outer + 3 * inner + outer
    kept = (rows * (inner + outer) * 33) // 32 if case["bits"] else rows * (inner + outer) * size
    if not case["backward"]:   # x and the parameters in; y, the statistics and the values of what is kept out
        values = rows * (inner + outer) if case["bits"] else rows * outer
        return {"bytes": (2 * rows * inner + weights + values) * size + 8 * rows, "flops": 2 * product}
    return {"bytes": (2 * rows * inner + 2 * weights) * size + kept + 8 * rows, "flops": 4 * product}


# -- in 64 bits -----------------------------------------------------------------
_LIBRARY = {"none": lambda z: z, "relu": F.relu, "gelu": F.gelu, "gelu_tanh": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}


def _kept_exactly(x):
    """The 8-bit form's value of each entry, from its definition."""
    rows, cols = x.shape
    size = F.pad(x.abs(), (0, -cols % BLOCK)).unflatten(1, (-1, BLOCK)).amax(2)
    e = torch.ceil(torch.log2(size / 127)).clamp(min=-127)
    e = torch.where(torch.exp2(e - 1) * 127 >= size, e - 1, e).clamp(min=-127)    # the logarithm may be off by one ulp
    e = torch.where(torch.exp2(e) * 127 < size, e + 1, e)
    step = torch.exp2(e).repeat_interleave(BLOCK, 1)[:, :cols]
    return (x / step).round() * step


def exact(case, seed):
    s = prepare(case, seed)
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    act = _LIBRARY[case["act"]] if "act" in case else None

    def want(*names):
        return [d[n].requires_grad_() for n in names]

    if case["op"] == "norm":
        x, w, b = want("x", "w", "b")
        y = F.layer_norm(x, x.shape[1:], w, b, EPS)
        var, mean = torch.var_mean(x.detach(), 1, correction=0)
        out = {"y": y.detach(), "mean": mean, "rstd": (var + EPS) ** -0.5}
        if case["train"]:
            out["dx"], out["dw"], out["db"] = torch.autograd.grad(y, (x, w, b), d["dy"])
        return out
    if case["op"] == "linear":
        x, w, b = want("x", "w", "b")
        z = F.linear(x, w, b)
        at = (_kept_exactly(z.detach()) if case["bits"] and case["train"] else z.detach()).requires_grad_()
        y = act(z.detach())
        out = {"y": y + d["r"] if case["residual"] else y}
        if case["train"]:
            dz, = torch.autograd.grad(act(at), at, d["dy"])
            out["dx"], out["dw"], out["db"] = torch.autograd.grad(z, (x, w, b), dz)
        return out
    if case["op"] == "keep":
        x = _kept_exactly(d["x"]).requires_grad_()
        dz, = torch.autograd.grad(act(x), x, d["dy"])
        return {"x": x.detach(), "dz": dz, "db": dz.sum(0)}
    if not case["backward"]:
        x = d["x"]
        z = F.linear(F.layer_norm(x, x.shape[1:], d["g"], d["b"], EPS), d["w1"], d["b1"])
        var, mean = torch.var_mean(x, 1, correction=0)
        out = {"y": F.linear(act(z), d["w2"], d["b2"]) + x, "mean": mean, "rstd": (var + EPS) ** -0.5}
        if case["bits"]:   # at the edge of a step, the last bit of a product's operand decides z's code: it has no one value
            out.update(x=_kept_exactly(x), z=None)
        else:
            out["z"] = z
        return out
    if case["bits"]:
        for name in ("x", "z"):
            q, e = s[name + "q"], s[name + "e"]
            step = torch.exp2(e.double() - 127).repeat_interleave(BLOCK, 1)[:, :q.shape[1]]
            d[name] = q.double() * step
    x, z, g, b, w1, w2 = want("x", "z", "g", "b", "w1", "w2")
    mean, rstd, dy = d["mean"][:, None], d["rstd"][:, None], d["dy"]
    # the layers' own vector-Jacobian products, joined by hand: each layer is read at what was kept of its input
    h = act(z)
    dh, dw2 = torch.autograd.grad(h @ w2.t(), (h, w2), dy, retain_graph=True)
    dz, = torch.autograd.grad(h, z, dh)
    a = ((x - mean) * rstd * g + b).detach().requires_grad_()
    da, dw1 = torch.autograd.grad(a @ w1.t(), (a, w1), dz)
    xh = ((x - mean) * rstd).detach()
    t = da * g.detach()
    dx = rstd * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True)) + dy
    return {"dx": dx.detach(), "dg": (da * xh).sum(0), "db": da.sum(0), "dw1": dw1, "db1": dz.sum(0), "dw2": dw2, "db2": dy.sum(0)}
