"""Float64 restatements of the expert products and of MXFP4 (OCP microscaling
formats v1.0), from their formulas, in numpy. The package has no reference
counterpart for these; their bounds are derived beside the tests.

* ``grouped_linear`` and its gradients: one product for each expert's rows.
* ``mxfp4_quant`` / ``mxfp4_values``: the block's scale from ``numpy.frexp``, the
  code as the nearest of the eight magnitudes, ties to the even code.
"""

from __future__ import annotations

import numpy as np

MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BLOCK = 32


def grouped_linear(x: np.ndarray, weight: np.ndarray, offsets: np.ndarray) -> np.ndarray:
    y = np.zeros((x.shape[0], weight.shape[1]))
    for e in range(weight.shape[0]):
        rows = slice(offsets[e], offsets[e + 1])
        y[rows] = x[rows].astype(np.float64) @ weight[e].astype(np.float64).T
    return y


def grouped_linear_grad_input(grad_y: np.ndarray, weight: np.ndarray, offsets: np.ndarray) -> np.ndarray:
    return grouped_linear(grad_y, weight.transpose(0, 2, 1), offsets)


def grouped_linear_grad_weight(grad_y: np.ndarray, x: np.ndarray, offsets: np.ndarray) -> np.ndarray:
    pairs = [(grad_y[a:b].astype(np.float64), x[a:b].astype(np.float64)) for a, b in zip(offsets[:-1], offsets[1:])]
    return np.stack([g.T @ v for g, v in pairs])


def mxfp4_quant(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """float [..., K] -> codes uint8 [..., 16 ceil(K / 32)], scale bytes uint8 [..., ceil(K / 32)]."""
    k = x.shape[-1]
    blocks = -(-k // BLOCK)
    v = np.zeros((*x.shape[:-1], blocks * BLOCK))
    v[..., :k] = x
    v = v.reshape(*x.shape[:-1], blocks, BLOCK)
    bad = ~np.isfinite(v).all(-1)
    v = np.where(bad[..., None], 0.0, v)
    amax = np.abs(v).max(-1)
    # amax = m 2^e, m in [0.5, 1): floor(log2 amax) = e - 1
    power = np.where(amax > 0, np.frexp(amax)[1] - 3, -127).clip(-127, 127)
    a = np.abs(v) / np.exp2(power)[..., None]
    above = np.searchsorted(MAGNITUDES, a, side="left").clip(0, 7)  # first magnitude >= a
    below = np.maximum(above - 1, 0)
    up, down = MAGNITUDES[above] - a, a - MAGNITUDES[below]
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)) | (a >= 6), above, below)
    code = np.where(np.signbit(v), code + 8, code).astype(np.uint8).reshape(*x.shape[:-1], blocks * BLOCK)
    scale = np.where(bad, 255, power + 127).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def mxfp4_values(codes: np.ndarray, scales: np.ndarray, width: int) -> np.ndarray:
    c = np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], -1)
    v = np.where(c >= 8, -1.0, 1.0) * MAGNITUDES[c & 7]
    scale = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * np.repeat(scale, BLOCK, axis=-1))[..., :width]
