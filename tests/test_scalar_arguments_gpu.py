"""Tensors without dimensions in place of the decode step's arguments: each call ends in
the refusal of the validating function."""

from __future__ import annotations

import pytest
import torch

from custom_cuda_kernals_amd import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("op", ["rope_at", "rope_to_cache", "paged_attention", "fp8_block_linear"])
def test_scalars_are_refused(op):
    x = torch.randn(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    cache = [torch.zeros(2, 16, 4, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    at, frequencies = torch.arange(3, device="cuda"), K.rope_frequencies(64)[0]
    codes, scale = K.fp8_quant(x.flatten(1), "e4m3", "block")
    args = {"rope_at": (x, x.clone(), at, frequencies),
            "rope_to_cache": (x, x.clone(), x.clone(), *cache, at, at, frequencies),
            "paged_attention": (x, *cache, torch.zeros(3, 1, dtype=torch.int64, device="cuda"), at),
            "fp8_block_linear": (codes, scale, codes, scale)}[op]
    getattr(K, op)(*args)
    for i, arg in enumerate(args):
        scalar = torch.zeros((), device="cuda").to(arg.dtype)
        with pytest.raises(ValueError):
            getattr(K, op)(*args[:i], scalar, *args[i + 1:])
