"""Plain 64-bit restatement of dropout's numbers, of the RMSNorm of a
residual's sum and of the rotation by positions on several axes (no counterpart
in the reference; parity unpinned).

Dropout's generator is Philox4x32-10 as Salmon, Moraes, Dror and Shaw define it
("Parallel random numbers: as easy as 1, 2, 3", 2011), in Python's and numpy's
unsigned integers.
"""
from __future__ import annotations

from typing import Sequence

import numpy as np
import torch

LOW = 2 ** 32 - 1


def philox(counter: Sequence, key: Sequence[int]):
    """Four words of a counter of four 32-bit words (ints or uint64 arrays)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & LOW, (a >> 32) ^ c[3] ^ k[1], a & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return c


def numbers(rows: int, hidden: int, seed: int, offset: int = 0, first_row: int = 0) -> torch.Tensor:
    """The 16-bit number of every value of rows first_row ..., int32 [rows, hidden]."""
    per = (hidden + 7) // 8
    low, half = np.uint64(LOW), np.uint64(32)
    block = np.arange(rows * per, dtype=np.uint64) + np.uint64(first_row * per)
    full = lambda v: np.full(rows * per, v, dtype=np.uint64)  # noqa: E731
    c = [block & low, block >> half, full(offset & LOW), full(offset >> 32)]
    k = [seed & LOW, seed >> 32 & LOW]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    u = np.stack([w for word in c for w in (word & np.uint64(0xFFFF), word >> np.uint64(16))], -1)
    return torch.from_numpy(u.astype(np.int32).reshape(rows, per * 8)[:, :hidden])


def factors(shape, p: float, seed: int, offset: int = 0) -> torch.Tensor:
    """What every value of a tensor of `shape` is multiplied with, float64."""
    hidden = shape[-1]
    rows = int(np.prod(shape[:-1], dtype=np.int64))
    t = round(p * 65536)
    kept = numbers(rows, hidden, seed, offset) >= t
    return (kept.double() * (65536 / (65536 - t) if t < 65536 else 0.0)).reshape(shape)


def rmsnorm(h: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5) -> torch.Tensor:
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * weight


def pair_axes(sections: Sequence[int], dealt: bool = False) -> list:
    """The axis of every pair: sections[0] pairs of axis 0, then axis 1's, ...; or
    dealt to the axes in turn while they have some left, the rest to axis 0."""
    if not dealt:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    n = len(sections)
    return [p % n if p // n < sections[p % n] else 0 for p in range(sum(sections))]


def columns(cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, sections: Sequence[int],
            dealt: bool = False):
    """The table rows [tokens, rotary / 2] that tokens at positions [axes, tokens]
    turn by: pair p from its axis's row."""
    axes = pair_axes(sections, dealt)
    pick = lambda t: torch.stack([t[positions[a].long(), p] for p, a in enumerate(axes)], -1)  # noqa: E731
    return pick(cos), pick(sin)


def rotate(x: torch.Tensor, c: torch.Tensor, s: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """x [tokens, heads, D] turned by the table rows c, s [tokens, R / 2] of its tokens."""
    half = c.shape[-1]
    c, s = c.to(x.dtype).unsqueeze(1), s.to(x.dtype).unsqueeze(1)
    cols = list(x.unbind(-1))
    for p in range(half):
        lo, hi = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
        a, b = cols[lo], cols[hi]
        cols[lo], cols[hi] = a * c[..., p] - b * s[..., p], b * c[..., p] + a * s[..., p]
    return torch.stack(cols, -1)
