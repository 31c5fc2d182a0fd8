"""Linear layers of a mixture-of-experts FFN on rows in expert order, and their
gradients: matrix products grouped by expert, with groups of any size.

An addition. ``offsets`` is what ``compute_permutation(...,
return_offsets=True)`` returns: rows ``offsets[e] .. offsets[e + 1]`` belong to
expert ``e``. The sizes stay on the GPU; nothing waits for them. Like the other
ops, these record nothing for autograd: a training step calls the two gradients.
"""

from __future__ import annotations

import torch

from custom_cuda_kernals_amd._lib import native

__all__ = ["grouped_linear", "grouped_linear_grad_input", "grouped_linear_grad_weight"]


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``y[s] = x[s] @ weight[e].T`` for each row ``s`` of expert ``e``.

    x: ``[S, K]``, weight: ``[E, N, K]``, contiguous device tensors of one dtype
    (float32 / float16 / bfloat16); offsets: int64 ``[E + 1]``, not decreasing,
    ``E <= 1024``. Sums are float32. Returns y ``[S, N]``, zeros in the rows before
    ``offsets[0]`` and from ``offsets[E]`` on.
    """
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.grouped_linear_call(x, weight, offsets)
    if out is not None:
        return out
    _check_dims(x, weight, 2, 3)
    y = torch.empty((x.shape[0], weight.shape[1]), dtype=x.dtype, device=x.device)
    native.grouped_linear_fwd(x, weight, offsets, y)
    return y


def grouped_linear_grad_input(grad_y: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """The gradient of ``grouped_linear``'s x: ``grad_x[s] = grad_y[s] @ weight[e]``.

    grad_y: ``[S, N]``; weight, offsets and dtypes as there. Returns ``[S, K]``,
    zeros in the rows of no expert."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.grouped_linear_grad_input_call(grad_y, weight, offsets)
    if out is not None:
        return out
    _check_dims(grad_y, weight, 2, 3)
    grad_x = torch.empty((grad_y.shape[0], weight.shape[2]), dtype=grad_y.dtype, device=grad_y.device)
    native.grouped_linear_grad_input(grad_y, weight, offsets, grad_x)
    return grad_x


def grouped_linear_grad_weight(grad_y: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """The gradient of ``grouped_linear``'s weight: ``grad_weight[e]`` is the sum of
    ``outer(grad_y[s], x[s])`` over the rows ``s`` of expert ``e``, zeros for an
    expert without rows.

    grad_y: ``[S, N]``, x: ``[S, K]``; offsets and dtypes as there. Returns
    ``[E, N, K]``."""
    # The ordinary call in one native call; None: the long way below, which raises the errors.
    out = native.grouped_linear_grad_weight_call(grad_y, x, offsets)
    if out is not None:
        return out
    _check_dims(grad_y, x, 2, 2)
    shape = (max(offsets.numel() - 1, 0), grad_y.shape[1], x.shape[1])
    grad_weight = torch.empty(shape, dtype=grad_y.dtype, device=grad_y.device)
    native.grouped_linear_grad_weight(grad_y, x, offsets, grad_weight)
    return grad_weight


def _check_dims(a: torch.Tensor, b: torch.Tensor, a_dims: int, b_dims: int) -> None:
    """What the output's shape is read from."""
    if a.dim() != a_dims or b.dim() != b_dims:
        raise ValueError(f"shape mismatch: expected tensors of {a_dims} and {b_dims} dimensions, got "
                         f"{tuple(a.shape)} and {tuple(b.shape)}")
