"""PagedCache.allocate makes its tensors in their own type: a cache is sized to fill the
card, so nothing larger may be made on the way."""

from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from custom_cuda_kernals_amd.llama_block import LlamaBlockConfig, PagedCache


class Made(TorchDispatchMode):
    """Bytes of every tensor that an operator returns."""

    def __init__(self):
        super().__init__()
        self.bytes = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        out = func(*args, **(kwargs or {}))
        if isinstance(out, torch.Tensor):
            self.bytes.append(out.untyped_storage().nbytes())
        return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float8_e4m3fn, torch.float8_e5m2])
def test_nothing_larger_than_the_cache(dtype):
    cfg = LlamaBlockConfig(num_heads=4, num_kv_heads=2, hidden_size=64)
    with Made() as made:
        cache = PagedCache.allocate(cfg, 3, 100, 16, dtype, "cpu", 0.5, 0.25)
    for t in (cache.keys, cache.values):
        assert t.shape == (21, 16, 2, 16) and t.dtype == dtype and not t.float().any()
    assert cache.keys.data_ptr() != cache.values.data_ptr()
    assert max(made.bytes) == cache.keys.untyped_storage().nbytes()
    assert cache.page_table.flatten().tolist() == list(range(21)) and cache.lengths.tolist() == [0, 0, 0]
    assert (cache.key_scale, cache.value_scale) == (0.5, 0.25)
