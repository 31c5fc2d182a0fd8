"""The decode step's operators in float64: rotary positions, FP8 values of a cache, the
attention of one token a sequence over a paged cache, and products of FP8 codes with a
scale for each block of 128."""

from __future__ import annotations

import numpy as np

from oracle import fp8 as ofp8

TILE = 128


def rope_at(x, positions, frequencies, layout="half", scale=1.0, inverse=False):
    """x [..., heads, D] in float64, positions [...], frequencies [R / 2]."""
    x = np.array(x, dtype=np.float64)
    half = len(frequencies)
    angle = np.asarray(positions, dtype=np.float64)[..., None, None] * np.asarray(frequencies, dtype=np.float64)
    c, s = scale * np.cos(angle), scale * np.sin(angle) * (-1.0 if inverse else 1.0)
    first = slice(0, half) if layout == "half" else slice(0, 2 * half, 2)
    second = slice(half, 2 * half) if layout == "half" else slice(1, 2 * half, 2)
    a, b = x[..., first].copy(), x[..., second].copy()
    x[..., first], x[..., second] = a * c - b * s, b * c + a * s
    return x


def paged_attention(q, keys, values, table, lengths, scale=None, window=0):
    """q [B, Hq, D], keys and values [pages, page, Hkv, D], all float64; (out, lse, the sum of p |v|, and
    the largest sum of |scale q k|, both for error bounds)."""
    b, heads, dim = q.shape
    pages, page, kv = keys.shape[:3]
    scale = dim ** -0.5 if scale is None else scale
    out, spread = np.zeros(q.shape), np.zeros(q.shape)
    lse, size = np.full((b, heads), -np.inf), np.zeros((b, heads))
    for i in range(b):
        n = min(max(int(lengths[i]), 0), table.shape[1] * page)
        at = np.arange(max(0, n - window) if window else 0, n)
        at = at[(table[i, at // page] >= 0) & (table[i, at // page] < pages)]
        if len(at) == 0:
            continue
        k, v = (c[table[i, at // page], at % page] for c in (keys, values))
        for h in range(heads):
            kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
            s = kh @ q[i, h] * scale
            p = np.exp(s - s.max())
            lse[i, h] = s.max() + np.log(p.sum())
            p /= p.sum()
            out[i, h], spread[i, h] = p @ vh, p @ np.abs(vh)
            size[i, h] = (np.abs(kh) @ np.abs(q[i, h])).max() * abs(scale)
    return out, lse, spread, size


def block_values(codes, scales, fmt, tall):
    """Values of codes (uint8 [..., M, K]); scales [..., M or ceil(M / 128), ceil(K / 128)], `tall` the latter."""
    v = ofp8.decode(codes, fmt).astype(np.float64)
    m, k = v.shape[-2:]
    s = np.repeat(scales.astype(np.float64), TILE, axis=-1)[..., :k]
    return v * (np.repeat(s, TILE, axis=-2)[..., :m, :] if tall else s)


def quant_group(x, fmt):
    """Codes and scales [M, ceil(N / 128)] of float32 x, one scale for 128 neighbours of a row."""
    m, n = x.shape
    codes, scales = np.empty((m, n), dtype=np.uint8), np.empty((m, -(-n // TILE)), dtype=np.float32)
    for j in range(scales.shape[1]):
        part = np.ascontiguousarray(x[:, j * TILE:(j + 1) * TILE])
        codes[:, j * TILE:(j + 1) * TILE], scales[:, j] = ofp8.quant_token(part, fmt)
    return codes, scales
