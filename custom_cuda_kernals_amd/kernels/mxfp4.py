"""MXFP4, the 4-bit microscaling format (OCP microscaling formats v1.0):
quantisation, its inverse, and the matrix product on gfx950's scaled MFMA, dense
or grouped by expert. An addition.

A tensor ``[..., K]`` is a pair ``(codes, scales)``:

* codes: uint8 ``[..., 16 * ceil(K / 32)]``, two e2m1 codes (0, 0.5, 1, 1.5, 2, 3,
  4, 6 and a sign) a byte, the lower element in the lower half; a row's last block
  of 32 is filled up with zeros;
* scales: float8_e8m0fnu ``[..., ceil(K / 32)]``, one power of two for 32
  neighbours: ``2 ** (floor(log2(max |x|)) - 2)``, at least ``2 ** -127``; NaN for a
  block with a NaN or an infinity.

``token_gather`` moves rows of codes and of scales as it moves FP8 rows: pass
``codes.view(torch.float8_e4m3fn)``, and view the result as it was.
"""

from __future__ import annotations

import torch

from custom_cuda_kernals_amd._lib import native

__all__ = ["mxfp4_quant", "mxfp4_dequant", "mxfp4_linear"]

_BLOCK = 32


def mxfp4_quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Quantise ``[..., K]`` (contiguous float32 / float16 / bfloat16 device tensor)
    along its last dimension: each element divided by its block's scale and rounded
    to the nearest e2m1 value, ties to the even code, beyond 6 to 6. Returns
    ``(codes, scales)``."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.mxfp4_quant_call(x)
    if out is not None:
        return out
    if x.dim() < 1:
        raise ValueError("shape mismatch: x must have at least 1 dimension")
    blocks = -(-x.shape[-1] // _BLOCK)
    codes = torch.empty((*x.shape[:-1], 16 * blocks), dtype=torch.uint8, device=x.device)
    scales = torch.empty((*x.shape[:-1], blocks), dtype=torch.float8_e8m0fnu, device=x.device)
    native.mxfp4_quant_fwd(x, codes, scales)
    return codes, scales


def mxfp4_dequant(codes: torch.Tensor, scales: torch.Tensor, width: int, dtype: torch.dtype = torch.bfloat16
                  ) -> torch.Tensor:
    """The values ``code * scale`` of the first ``width`` elements of each row
    (``ceil(width / 32)`` blocks), rounded once to ``dtype``. Returns
    ``[..., width]``."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.mxfp4_dequant_call(codes, scales, width, dtype)
    if out is not None:
        return out
    if codes.dim() < 1 or width < 0:
        raise ValueError(f"shape mismatch: codes must have at least 1 dimension and width be >= 0, got "
                         f"{tuple(codes.shape)} and {width}")
    values = torch.empty((*codes.shape[:-1], width), dtype=dtype, device=codes.device)
    native.mxfp4_dequant_fwd(codes, scales, values)
    return values


def mxfp4_linear(x_codes: torch.Tensor, x_scales: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor,
                 offsets: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``y = x @ w.T`` of two MXFP4 operands, sums in float32.

    x: codes ``[S, 16 * B]`` and scales ``[S, B]``. Without offsets w is ``[N, ...]``;
    with offsets (int64 ``[E + 1]``, as for ``grouped_linear``) w is ``[E, N, ...]``
    and row ``s`` of expert ``e`` meets ``w[e]``, rows of no expert being zeros.
    Returns y ``[S, N]`` of ``out_dtype`` (float32 / float16 / bfloat16)."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.mxfp4_linear_call(x_codes, x_scales, w_codes, w_scales, offsets, out_dtype)
    if out is not None:
        return out
    if x_codes.dim() != 2 or w_codes.dim() != (2 if offsets is None else 3):
        raise ValueError(f"shape mismatch: x_codes must be 2-D and w_codes {2 if offsets is None else 3}-D, got "
                         f"{tuple(x_codes.shape)} and {tuple(w_codes.shape)}")
    y = torch.empty((x_codes.shape[0], w_codes.shape[-2]), dtype=out_dtype, device=x_codes.device)
    native.mxfp4_linear_fwd(x_codes, x_scales, w_codes, w_scales, offsets, y)
    return y
