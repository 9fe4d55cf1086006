"""Plain PyTorch statement of the feed-forward operators.

Layer norm, the linear layer with activation and residual, and the 8-bit form of
an activation: what CPU tensors run and what the kernels are tested against.
Everything is computed in f32 (f64 for f64 inputs) and rounded once, to the
inputs' type.  Matrices are [rows, cols]; nothing here is meant to be fast.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

BLOCK = 32          # columns that share an exponent in the 8-bit form
NAN_BYTE = 255      # exponent byte of a block that held a NaN or an infinity


def wide(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.float64 else t.float()


def act(name: str, z: torch.Tensor) -> torch.Tensor:
    if name == "none":
        return z
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z / (1 + torch.exp(-z))


def act_slope(name: str, z: torch.Tensor) -> torch.Tensor:
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z ** 3))
        t = z * (1 - th * th)      # 0 before z^2 leaves the type's range
        return 0.5 * (1 + th) + 0.5 * c * (t + 3 * 0.044715 * (t * z * z))
    sg = torch.sigmoid(z)
    return sg * (1 + z * (1 - sg))


def norm_forward(x, w, b, eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    v = wide(x)
    mean = v.mean(1)
    c = v - mean[:, None]
    rstd = 1 / torch.sqrt((c * c).mean(1) + eps)
    y = c * rstd[:, None]
    if w is not None:
        y = y * wide(w)
    if b is not None:
        y = y + wide(b)
    return y.to(x.dtype), mean, rstd


def norm_backward(dy, x, mean, rstd, w, add) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    g = wide(dy)
    xh = (wide(x) - mean[:, None]) * rstd[:, None]
    t = g if w is None else g * wide(w)
    dx = rstd[:, None] * (t - t.mean(1, keepdim=True) - xh * (t * xh).mean(1, keepdim=True))
    if add is not None:
        dx = dx + wide(add)
    return dx.to(dy.dtype), (g * xh).sum(0).to(dy.dtype), g.sum(0).to(dy.dtype)


def keep8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(codes [rows, cols] int8, exponent bytes [rows, blocks] uint8)."""
    rows, cols = x.shape
    v = F.pad(wide(x), (0, -cols % BLOCK)).view(rows, -(-cols // BLOCK), BLOCK)
    most = v.abs().amax(2)
    bad = ~torch.isfinite(v).all(2)
    mantissa, exponent = torch.frexp(torch.where(bad, torch.ones_like(most), most))
    e = torch.where(mantissa > 127 / 128, exponent - 6, exponent - 7)    # most <= 127 * 2^e
    e = torch.where(mantissa == 0, torch.full_like(e, -127), e).clamp(min=-127)
    q = torch.round(torch.ldexp(v, -e[..., None]))
    last = (e == 122)[..., None]                                         # 64 * 2^122 would be an infinity
    q = torch.where(last, q.clamp(-63, 63), q)
    q = torch.where(bad[..., None], torch.zeros_like(q), q).to(torch.int8)
    byte = torch.where(bad, torch.full_like(e, NAN_BYTE), e + 127).to(torch.uint8)
    return q.flatten(1)[:, :cols].contiguous(), byte


def values8(q: torch.Tensor, e: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    rows, cols = q.shape
    v = F.pad(q.to(dtype), (0, -cols % BLOCK)).view(rows, -(-cols // BLOCK), BLOCK)
    v = torch.ldexp(v, e.int()[..., None] - 127)
    v = torch.where((e == NAN_BYTE)[..., None], torch.full_like(v, math.nan), v)
    return v.flatten(1)[:, :cols].contiguous()


def restore8(q: torch.Tensor, e: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What the codes stand for, in ``dtype``; in f16 what would be 65536 is the largest number."""
    v = values8(q, e, torch.float64 if dtype == torch.float64 else torch.float32)
    return (v.clamp(-65504, 65504) if dtype == torch.float16 else v).to(dtype)


def linear_forward(x, w, b, name: str, residual) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, z); z unrounded."""
    z = wide(x) @ wide(w).t()
    if b is not None:
        z = z + wide(b)
    y = act(name, z)
    if residual is not None:
        y = y + wide(residual)
    return y.to(x.dtype), z


def act_backward(dy, z: Optional[torch.Tensor], name: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dz unrounded, its sum over the rows)."""
    dz = wide(dy) if name == "none" else wide(dy) * act_slope(name, wide(z))
    return dz, dz.sum(0)
