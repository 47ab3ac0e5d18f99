"""Restatement of the quantized key / value cache and of the attention over its pages: float32 numpy in the order of the
definition for codes, scales and zero points, float64 for attention.  Test infrastructure only."""

from __future__ import annotations

import numpy as np

F = np.float32


def grid(bits: int) -> tuple[int, int]:
    return -(1 << (bits - 1)), (1 << (bits - 1)) - 1


def quantize(x, bits: int, symmetric: bool):
    """``(code - qmin as uint8, scale, zero)`` of rows of float32 along the last axis."""
    x = np.asarray(x, F)
    qmin, qmax = grid(bits)
    with np.errstate(all="ignore"):
        lo, hi = np.minimum(x.min(-1), F(0)), np.maximum(x.max(-1), F(0))  # (both keep a NaN)
        if symmetric:
            scale = np.maximum(np.maximum(np.abs(lo), np.abs(hi)) / F((qmax - qmin) / 2), F(1e-8))
            zero = np.zeros_like(scale)
        else:
            scale = np.maximum((hi - lo) / F(qmax - qmin), F(1e-8))
            zero = np.clip(F(qmin) - np.rint(lo / scale), F(qmin), F(qmax))
        c = np.clip(np.rint(x / scale[..., None]) + zero[..., None], F(qmin), F(qmax))
    return (np.where(np.isnan(c), 0, c).astype(np.int32) - qmin).astype(np.uint8), scale, zero


def pack(u, bits: int):
    return u if bits == 8 else u[..., 0::2] | u[..., 1::2] << 4


def unpack(b, bits: int):
    b = np.asarray(b).view(np.uint8)
    return b if bits == 8 else np.stack((b & 15, b >> 4), -1).reshape(*b.shape[:-1], -1)


def values(codes, scale, zero, bits: int):
    """float32 ``(code - zero) * scale`` of packed rows."""
    z = np.zeros_like(scale) if zero is None else zero
    with np.errstate(invalid="ignore"):
        return (unpack(codes, bits).astype(F) + F(grid(bits)[0]) - z[..., None]) * scale[..., None]


def attention(q, k_pages, v_pages, table, q_starts, kv_lens, scale, causal=True, window=None):
    """float64 result for ``q`` (tokens, heads, dim) over pages ``(pages, kv_heads, page_size, dim)``."""
    q = np.asarray(q, np.float64)
    pages, kv_heads, page_size, _ = k_pages.shape
    group = q.shape[1] // kv_heads
    out = np.zeros(q.shape)
    for b in range(len(kv_lens)):
        lo, hi = int(q_starts[b]), int(q_starts[b + 1])
        length = max(0, min(int(kv_lens[b]), table.shape[1] * page_size))
        j = np.arange(length)
        page = table[b][j // page_size] if length else np.zeros(0, int)
        known = (page >= 0) & (page < pages)
        j, page = j[known], page[known]
        k, v = (p[page, :, j % page_size].astype(np.float64) for p in (k_pages, v_pages))
        for i in range(lo, hi):
            place = length - (hi - lo) + (i - lo)
            seen = (j <= place) if causal else np.ones(len(j), bool)
            if window is not None:
                seen &= j > place - window
            if not seen.any():
                continue
            for h in range(q.shape[1]):
                s = k[seen, h // group] @ q[i, h] * scale
                p = np.exp(s - s.max())
                out[i, h] = p @ v[seen, h // group] / p.sum()
    return out
