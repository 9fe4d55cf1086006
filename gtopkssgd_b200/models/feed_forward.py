"""Residual feed-forward block over sequences, on the framework's own kernels
(``ops/feed_forward.py``): y = x + W2 act(W1 norm(x) + b1) + b2."""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from ..ops.activation8 import act_of, bits_of
from ..ops.feed_forward import feed_forward_block


class FeedForward(nn.Module):
    """``bits=8``: the backward pass reads 8-bit copies of the block's input and of
    the activation's input, a quarter of f32's bytes.  ``compute_dtype``: the type
    the block computes in (None: the parameters'); the parameters, their gradients
    and the block's input and output keep their own."""

    def __init__(self, dim: int, hidden: int, activation: str = "gelu", eps: float = 1e-5, bits: int = 0, compute_dtype=None):
        super().__init__()
        if act_of(activation) == 0:
            raise ValueError("a feed-forward block has an activation")
        self.activation, self.eps, self.bits, self.compute_dtype = activation, eps, bits_of(bits), compute_dtype
        self.norm_weight = nn.Parameter(torch.ones(dim))
        self.norm_bias = nn.Parameter(torch.zeros(dim))
        self.w1 = nn.Parameter(torch.empty(hidden, dim).uniform_(-1 / math.sqrt(dim), 1 / math.sqrt(dim)))
        self.b1 = nn.Parameter(torch.zeros(hidden))
        self.w2 = nn.Parameter(torch.empty(dim, hidden).uniform_(-1 / math.sqrt(hidden), 1 / math.sqrt(hidden)))
        self.b2 = nn.Parameter(torch.zeros(dim))

    def forward(self, x):
        dtype = self.compute_dtype or self.w1.dtype
        args = [t.to(dtype) for t in (x, self.norm_weight, self.norm_bias, self.w1, self.b1, self.w2, self.b2)]
        return feed_forward_block(*args, self.activation, self.eps, self.bits).to(x.dtype)

    def extra_repr(self) -> str:
        return "dim=%d, hidden=%d, activation=%s, bits=%d" % (self.w2.size(0), self.w1.size(0), self.activation, self.bits)
