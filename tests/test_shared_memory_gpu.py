"""The Python calls refuse what test_shared_memory_cpu.py refuses of the binding: no launch
is made. Slices side by side of one projection go through, in place."""

from __future__ import annotations

import pytest
import torch

from custom_cuda_kernals_amd import kernels as K

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _refused(fn, *args, **kw):
    with pytest.raises(ValueError, match="are the same memory, or share some of it"):
        fn(*args, **kw)


def test_refusals():
    rows = torch.randn(9, 8, 64, device="cuda").to(BF16)
    was = rows.clone()
    positions, slots, (frequencies, _) = torch.arange(9, device="cuda"), torch.arange(9, device="cuda"), K.rope_frequencies(64)
    for q, k in ((rows[:, :5], rows[:, 4:6]), (rows[:, 4:6], rows[:, :5]), (rows, rows), (rows[:8], rows[1:])):
        n = len(q)
        _refused(K.rope_at, q, k, positions[:n], frequencies, inplace=True)
    cache = torch.zeros(2, 2, 16, 2, 64, dtype=BF16, device="cuda")
    q, k, v = rows[:, :4], rows[:, 4:6], rows[:, 6:]
    both = torch.zeros(3, 16, 2, 64, dtype=BF16, device="cuda")
    for keys, values in ((cache[0], cache[0]), (both[:2], both[1:]), (both[1:], both[:2])):
        for kw in ({}, {"inplace": True}):
            _refused(K.rope_to_cache, q, k, v, keys, values, slots, positions, frequencies, **kw)
    _refused(K.rope_to_cache, q, rows[:, 3:5], v, *cache, slots, positions, frequencies, inplace=True)
    _refused(K.rope_to_cache, q, k, rows[:, :2], *cache, slots, positions, frequencies, inplace=True)
    _refused(K.rope_to_cache, q, cache[0].view(32, 2, 64)[:9], v, *cache, slots, positions, frequencies)
    torch.cuda.synchronize()
    assert torch.equal(rows, was) and not cache.any() and not both.any()


def test_heads_in_turn_go_through():
    """q and k of one tensor, a head each in turn, and of one whose heads lie apart from each other by all tokens."""
    positions, (frequencies, _) = torch.arange(9, device="cuda"), K.rope_frequencies(64)
    x = torch.randn(9, 8, 64, device="cuda").to(BF16)
    want = K.rope_at(x[:, 0::2].contiguous(), x[:, 1::2].contiguous(), positions, frequencies)
    for y in (x.clone(), x.transpose(0, 1).contiguous().transpose(0, 1)):
        K.rope_at(y[:, 0::2], y[:, 1::2], positions, frequencies, inplace=True)
        assert torch.equal(y[:, 0::2], want[0]) and torch.equal(y[:, 1::2], want[1])
