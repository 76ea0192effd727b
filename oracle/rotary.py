"""CPU restatement of rotary positions as include/fused_attn.h defines them.  TEST INFRASTRUCTURE ONLY.

What pins each function (tests/test_rotary.py, on the CPU):
  frequencies  closed forms: no scaling is base^(-2j/D); a factor of 1 changes nothing; what turns often keeps its frequency, what turns
               seldom is divided, whole
  tables       position 0; the addition theorem over positions
  rotate       multiplication of complex numbers, an independent formulation; back and forth; the scalar product of two rotated
               vectors depends on the difference of their positions alone
"""
import math

import numpy as np
import torch


def frequencies(dims, base=10000.0, scaling="none", factor=1.0, original_rows=1.0, low=1.0, high=4.0):
    """float64 [dims / 2]: what a column turns by for each position."""
    j = np.arange(dims // 2, dtype=np.float64)
    if scaling == "base":
        base = base * factor ** (dims / (dims - 2.0))
    f = base ** (-2.0 * j / dims)
    if scaling == "linear":
        return f / factor
    if scaling == "turns":
        keep = np.clip((original_rows * f / (2 * np.pi) - low) / (high - low), 0, 1)
        return f * (keep + (1 - keep) / factor)
    if scaling == "index":
        index = [dims * math.log(original_rows / (2 * math.pi * t)) / (2 * math.log(base)) for t in (high, low)]
        a, b = max(math.floor(index[0]), 0), min(math.ceil(index[1]), dims - 1)
        keep = 1 - np.clip((j - a) / max(b - a, 0.001), 0, 1)
        return f * (keep + (1 - keep) / factor)
    return f


def tables(rows, dims, amplitude=1.0, **how):
    """cos and sin in float64, [rows, dims / 2]."""
    angle = np.arange(rows, dtype=np.float64)[:, None] * frequencies(dims, **how)[None]
    return amplitude * np.cos(angle), amplitude * np.sin(angle)


def rotate(x, cos, sin, positions, first=0, interleaved=False, inverse=False, exists=None):
    """x [B, L, heads, H] (16 bits) by the float32 tables' rows at positions [B, L], products and sums rounded to float32, the result to
    x's type; zeros where the position has no row or `exists` [B, L] is false."""
    rows, half = cos.shape
    ok = (positions >= 0) & (positions < rows)
    if exists is not None:
        ok &= exists
    at = positions.clamp(0, rows - 1).long()
    c, s = cos[at][:, :, None], sin[at][:, :, None]
    s = -s if inverse else s
    y = x.float()
    part = y[..., first:first + 2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    a, b = a * c - b * s, b * c + a * s                            # (eager operations: every one rounds)
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    y = torch.cat([y[..., :first], turned, y[..., first + 2 * half:]], -1)
    return torch.where(ok[:, :, None, None], y, 0.0).to(x.dtype)
