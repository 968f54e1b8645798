"""Plain 64-bit restatement of the 8-bit checkpoints of rows and of the
per-head norm of queries and keys with its rotation (no counterpart in the
reference; parity unpinned).

The format, from its definition: blocks of 32 values of a row; with a = max |x|
and M = 127 ("int8") or 448 ("e4m3"), e is the least integer with a <= M 2^e,
at least -100; a value is x 2^-e rounded to nearest even (to an integer, or to
an e4m3 number), times 2^e.  A block with a value that is not finite is NaN; a
value that rounds to 2^128 or more is infinite, as it is in bf16.
"""
from __future__ import annotations

import torch

MAX = {"int8": 127.0, "e4m3": 448.0}


def _split(x: torch.Tensor) -> torch.Tensor:
    C = x.shape[-1]
    pad = torch.zeros(*x.shape[:-1], -C % 32, dtype=torch.float64)
    return torch.cat([x.detach().cpu().double(), pad], -1).reshape(*x.shape[:-1], (C + 31) // 32, 32)


def exponents(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """e of every block, by search; 128 for a block that is not finite."""
    a = _split(x).abs().amax(-1)
    e = torch.full(a.shape, 128.0, dtype=torch.float64)
    for k in range(127, -101, -1):
        e = torch.where(a <= MAX[fmt] * 2.0 ** k, float(k), e)
    return torch.where(a.isfinite(), e, 128.0)


def quantised(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """The numbers held (integers, or e4m3 numbers), [..., blocks, 32]; zeros
    in a block that is not finite."""
    e = exponents(x, fmt).unsqueeze(-1)
    v = _split(x) * torch.exp2(-e)
    v = torch.where(e == 128.0, 0.0, v)
    if fmt == "int8":
        return torch.round(v)
    # e4m3: 3 bits after the leading one, exponents from -6 up, steps of 2^-9 below
    step = torch.full_like(v, 2.0 ** -9)
    for k in range(-5, 9):
        step = torch.where(v.abs() >= 2.0 ** k, 2.0 ** (k - 3), step)
    return torch.round(v / step) * step


def held(x: torch.Tensor, fmt: str) -> torch.Tensor:
    """The values a checkpoint of x stands for, float64 of x's shape."""
    if fmt is None:
        return x.detach().cpu().double()
    e = exponents(x, fmt).unsqueeze(-1)
    v = quantised(x, fmt) * torch.exp2(e)
    v = torch.where(v.abs() >= 2.0 ** 128, v * float("inf"), v)
    v = torch.where(e == 128.0, float("nan"), v)
    return v.flatten(-2)[..., :x.shape[-1]]


def qk_norm_rope(x: torch.Tensor, weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, eps: float = 1e-5,
                 interleaved: bool = False) -> torch.Tensor:
    """x [T, heads, D] with the table rows of its tokens, cos / sin [T, R/2];
    differentiable, in x's dtype."""
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(x.dtype)
    c, s = cos.to(x.dtype).unsqueeze(1), sin.to(x.dtype).unsqueeze(1)
    half = cos.shape[-1]
    cols = list(y.unbind(-1))
    for p in range(half):
        lo, hi = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
        a, b = cols[lo], cols[hi]
        cols[lo] = a * c[..., p] - b * s[..., p]
        cols[hi] = b * c[..., p] + a * s[..., p]
    return torch.stack(cols, -1)
