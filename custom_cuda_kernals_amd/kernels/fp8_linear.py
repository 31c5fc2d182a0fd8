"""Linear layers on FP8 codes with a scale for each block of 128 contracted elements: the
products of what ``fp8_quant`` writes with ``granularity="group"`` or ``"block"``. An
addition.

Their gradients are the same operator: a 128 x 128 tile stays one when its tensor is
transposed, so with a weight in ``"block"`` layout ::

    grad_x = fp8_block_linear(*fp8_quant(grad_y, "e5m2", "group"), w_codes.t().contiguous(),
                              w_scale.t().contiguous())

and with activations and ``grad_y`` in ``"block"`` layout too, ``grad_w =
fp8_block_linear(grad_codes.t().contiguous(), grad_scale.t().contiguous(),
x_codes.t().contiguous(), x_scale.t().contiguous())``.
"""

from __future__ import annotations

import torch

from custom_cuda_kernals_amd._lib import native

__all__ = ["fp8_block_linear"]


def fp8_block_linear(x_codes: torch.Tensor, x_scale: torch.Tensor, w_codes: torch.Tensor, w_scale: torch.Tensor,
                     offsets: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``y = dequant(x) @ dequant(w).T``.

    x: codes ``[S, K]`` (``float8_e4m3fn`` or ``float8_e5m2``, w's the same or the other)
    with scales ``[S, ceil(K / 128)]`` (``"group"``) or ``[ceil(S / 128), ceil(K / 128)]``
    (``"block"``). w: ``[N, K]`` with ``[ceil(N / 128), ceil(K / 128)]``; with offsets
    (int64 ``[E + 1]``, as for ``grouped_linear``) ``[E, N, K]`` with ``[E, ceil(N / 128),
    ceil(K / 128)]``, and row ``s`` of expert ``e`` meets ``w[e]``, rows of no expert being
    zeros. Returns y ``[S, N]`` of ``out_dtype`` (float32 / float16 / bfloat16).

    ``out_dtype`` chooses the sums. float32: of exact products, in float32. 16 bits: by the
    FP8 matrix instructions, which cut off what is below 2^-13 of the largest of eight
    neighbouring products, and in float32 beyond those eight. That is off by at most
    ``7 * 2^-13 * sum |x w|`` and usually by 1e-5 of that sum, which is not small beside a
    result whose products cancel. Where that matters, take float32 and round it."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.fp8_block_linear_call(x_codes, x_scale, w_codes, w_scale, offsets, out_dtype)
    if out is not None:
        return out
    if x_codes.dim() != 2 or w_codes.dim() != (2 if offsets is None else 3):
        raise ValueError(f"shape mismatch: x_codes must be 2-D and w_codes {2 if offsets is None else 3}-D, got "
                         f"{tuple(x_codes.shape)} and {tuple(w_codes.shape)}")
    y = torch.empty((x_codes.shape[0], w_codes.shape[-2]), dtype=out_dtype, device=x_codes.device)
    native.fp8_block_linear_fwd(x_codes, x_scale, w_codes, w_scale, offsets, y)
    return y
