"""Rotary positions of any kind: given positions, half-split or interleaved pairs,
part of a head, scaled for long contexts; and their gradient. An addition beside
``rope``, which turns whole heads by tables of the positions ``0 .. S - 1``.

A pair ``(a, b)`` of elements turns by ``angle = position * frequency`` of its pair::

    a' = scale * (a * cos(angle) - b * sin(angle))
    b' = scale * (b * cos(angle) + a * sin(angle))

The angles are formed in float64: off by 2**-51 of themselves, which is below the
results' other errors (2**-23) up to 2**28. Like the other ops, these record nothing for
autograd: the gradient is ``rope_at(..., inverse=True)`` of the outputs' gradients.
"""

from __future__ import annotations

import math

import torch

from custom_cuda_kernals_amd._lib import native

__all__ = ["rope_frequencies", "rope_at"]

SCALINGS = ("none", "linear", "ntk", "parts", "yarn")


def rope_frequencies(rotary_dim: int, theta: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                     original_length: int = 8192, low: float | None = None, high: float | None = None,
                     device: torch.device | str = "cuda") -> tuple[torch.Tensor, float]:
    """Angles a position and the scale of the turned elements, for a head of which
    ``rotary_dim`` elements turn: ``(frequencies float64 [rotary_dim / 2], scale)``.

    ``frequencies[i] = theta ** (-2 i / rotary_dim)``, and for contexts ``factor`` times
    as long as those of training:

    * ``"linear"``: divided by ``factor``;
    * ``"ntk"``: of ``theta * factor ** (rotary_dim / (rotary_dim - 2))``;
    * ``"parts"``: those that turn ``low`` (1) times or less within ``original_length``
      positions divided by ``factor``, those of ``high`` (4) or more as they are, and
      between them on the straight line between both;
    * ``"yarn"``: the same with ``high`` 32, and scale ``0.1 * ln(factor) + 1``. This is
      the published formula, straight in the number of turns. Checkpoints whose code is
      straight in the index of the pair instead, between the bounds' rounded indices, have
      other frequencies between both (up to 1.7 times these at theta 10**6, factor 4):
      make those, float64, and pass them to ``rope_at`` in place of these.
    """
    if rotary_dim < 0 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and not negative, got {rotary_dim}")
    if scaling not in SCALINGS:
        raise ValueError(f"scaling must be one of {SCALINGS}, got {scaling!r}")
    if not theta > 0 or not factor >= 1 or original_length < 1:
        raise ValueError(f"theta must be positive, factor and original_length at least 1, got {theta}, {factor} and "
                         f"{original_length}")
    if scaling == "ntk" and rotary_dim > 2:
        theta = theta * factor ** (rotary_dim / (rotary_dim - 2))
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    frequencies = theta ** (-i / max(rotary_dim, 1))
    if scaling == "linear":
        frequencies = frequencies / factor
    if scaling in ("parts", "yarn"):
        low = 1.0 if low is None else low
        high = (4.0 if scaling == "parts" else 32.0) if high is None else high
        if not high > low:
            raise ValueError(f"high must be above low, got {low} and {high}")
        turns = original_length * frequencies / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        frequencies = frequencies / factor * (1.0 - keep) + frequencies * keep
    return frequencies.to(device), 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0


def rope_at(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *,
            layout: str = "half", scale: float = 1.0, inverse: bool = False, inplace: bool = False
            ) -> tuple[torch.Tensor, torch.Tensor]:
    """Turn q ``[..., Hq, D]`` and k ``[..., Hkv, D]`` (float32 / float16 / bfloat16 device
    tensors of one dtype) to ``positions`` (int64 ``[...]``, one for each token).

    ``frequencies``: float64 ``[R / 2]``, ``R <= D <= 2048``; the elements of a head from
    R on are copied. ``layout``: pairs ``(x[i], x[i + R / 2])`` (``"half"``) or
    ``(x[2 i], x[2 i + 1])`` (``"interleaved"``). ``inverse`` turns by the negative angle:
    the gradient. q and k are contiguous, or ``[tokens, heads, D]`` with any strides of
    tokens and heads (slices of a projection's output). Returns contiguous tensors, or q
    and k with ``inplace=True``, when they have no elements in common."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.rope_at_call(q, k, positions, frequencies, layout, float(scale), inverse, inplace)
    if out is not None:
        return (q, k) if inplace else out
    if inplace:
        q_out, k_out = q, k
    else:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    native.rope_at_fwd(q, k, positions, frequencies, q_out, k_out, layout, float(scale), bool(inverse))
    return q_out, k_out
