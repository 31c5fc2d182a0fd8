"""A paged key-value cache and the attention of one new token a sequence over it. An
addition.

A cache is two tensors ``[pages, page_size, Hkv, D]``, keys and values, of the heads'
dtype or of FP8 codes (``float8_e4m3fn`` / ``float8_e5m2``) that stand for ``code *
scale`` with one scale for all keys and one for all values. A sequence's position ``t``
is at place ``t % page_size`` of page ``page_table[b, t // page_size]``; as a *slot* it
has the number ``page * page_size + place``. A page outside ``[0, pages)``, -1 for
instance, is one that the sequence does not have (any more): its positions are left out.
"""

from __future__ import annotations

import torch

from custom_cuda_kernals_amd._lib import native

__all__ = ["rope_to_cache", "paged_attention"]


def rope_to_cache(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_cache: torch.Tensor,
                  value_cache: torch.Tensor, slots: torch.Tensor, positions: torch.Tensor, frequencies: torch.Tensor, *,
                  layout: str = "half", scale: float = 1.0, key_scale: float = 1.0, value_scale: float = 1.0,
                  inplace: bool = False) -> torch.Tensor:
    """Turn q and k to their positions as ``rope_at`` does, and write k and v into the
    cache, in one launch; returns the turned q (q itself with ``inplace=True``).

    q ``[..., Hq, D]``, k and v ``[..., Hkv, D]``; ``slots``, ``positions``: int64 ``[...]``.
    A token whose slot is outside the cache (-1, say) is not written; no two tokens of a
    call may have the same slot, which then would hold parts of both. The caches share no
    memory with each other or with q, k and v, nor q with k or v in place. Without frequencies
    (``[0]``) nothing turns. Into an FP8 cache go codes of the values divided by
    ``key_scale`` / ``value_scale``, those beyond the format's largest value as that."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.rope_to_cache_call(q, k, v, key_cache, value_cache, slots, positions, frequencies, layout,
                                    float(scale), float(key_scale), float(value_scale), inplace)
    if out is not None:
        return q if inplace else out
    q_out = q if inplace else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    native.rope_to_cache_fwd(q, k, v, key_cache, value_cache, slots, positions, frequencies, q_out, layout,
                             float(scale), float(key_scale), float(value_scale))
    return q_out


def paged_attention(q: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, page_table: torch.Tensor,
                    lengths: torch.Tensor, *, scale: float | None = None, window: int = 0, key_scale: float = 1.0,
                    value_scale: float = 1.0, return_lse: bool = False
                    ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """``softmax(scale * q . k) . v`` of one token a sequence over its cached positions.

    q: ``[B, Hq, D]`` (float32 / float16 / bfloat16, D a multiple of 16, at most 256; any
    strides of sequences and heads), Hq a multiple of the cache's Hkv: query head h reads
    key-value head ``h // (Hq // Hkv)``. page_table: int64 ``[B, pages of each]``, lengths:
    int64 ``[B]``, the positions each sequence has, the new token's own among them (at
    most what its table holds is read). ``scale``: ``D ** -0.5`` unless given. ``window``:
    only the last so many positions (0: all). Scores, sums and the output's accumulators
    are float32.

    Returns out ``[B, Hq, D]`` of q's dtype, and with ``return_lse`` the logarithm of each
    head's sum of exponentials, float32 ``[B, Hq]``, by which outputs over parts of a
    context are joined. A sequence without positions: zeros, and -infinity. An infinite
    value that is seen makes its element infinite (NaN with one of the other sign, or where
    its weight is less than float32 has); sequences that hold such, or NaN, take longer."""
    dim = q.shape[-1] if q.dim() else 0
    scale = float(dim or 1) ** -0.5 if scale is None else float(scale)
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.paged_attention_call(q, key_cache, value_cache, page_table, lengths, scale, window, float(key_scale),
                                      float(value_scale), return_lse)
    if out is not None:
        return out
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    bytes_ = native.paged_attention_workspace(q, key_cache, page_table)
    workspace = torch.empty(bytes_ // 4, dtype=torch.float32, device=q.device)
    native.paged_attention_fwd(q, key_cache, value_cache, page_table, lengths, out, lse, workspace, scale, int(window),
                               float(key_scale), float(value_scale))
    return (out, lse) if return_lse else out
