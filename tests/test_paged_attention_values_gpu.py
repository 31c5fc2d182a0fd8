"""paged_attention where seen values are infinite, no numbers, or so large that their sum is
not a float32 while their average is: against the float64 formula, by which a position's
weight is never zero, so that an infinite value makes its element infinite, two of either
sign make it NaN, and nothing else changes. Bounds as in test_paged_attention_gpu.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from oracle import decode
from tests.test_paged_attention_gpu import DTYPES, IDS, U, _case, _wide

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")

def _check(q, keys, values, table, lengths, **kw):
    out, lse = K.paged_attention(q.cuda(), keys.cuda(), values.cuda(), table.cuda(), lengths.cuda(), return_lse=True, **kw)
    with np.errstate(invalid="ignore"):
        want, want_lse, spread, size = decode.paged_attention(q.double().numpy(), keys.double().numpy(),
                                                              values.double().numpy(), table.numpy(), lengths.numpy(),
                                                              kw.get("scale"))
    got = out.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    infinite = np.isinf(want)
    assert np.array_equal(np.isinf(got), infinite) and np.array_equal(got[infinite], want[infinite])
    longest = int(lengths.max())
    d = (q.shape[-1] + 4) * U * size
    info = torch.finfo(q.dtype)
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
        bound = ((2 * d + 2.0 ** -16 + (2 * longest + 128) * U)[..., None] * spread
                 + np.maximum(np.abs(want) * info.eps / 2, info.smallest_normal * info.eps / 2))
    fine = np.isfinite(want)
    assert (off[fine] <= bound[fine]).all()
    lse = lse.double().cpu().numpy()
    fine = np.isfinite(want_lse)
    assert np.array_equal(np.isfinite(lse), fine)
    # a float32 power of two up to 40 beside the sum's logarithm: 2^-19 of rounding, twice
    limit = d + (longest + 64) * U + np.abs(np.where(fine, want_lse, 0)) * 4 * U + 2.0 ** -18
    assert (np.abs(lse[fine] - want_lse[fine]) <= limit[fine]).all()
    return out


LENGTHS = {"short": [1, 17, 40, 60], "long": [2500, 31, 0, 1030]}


@pytest.mark.parametrize("pages", [0, 1, 30, 1000])
@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv,dim,cache", [(8, 2, 64, None), (32, 8, 128, None), (12, 4, 80, None), (2, 2, 256, None),
                                                (8, 2, 128, torch.float8_e5m2), (4, 4, 16, torch.float8_e5m2)])
def test_infinite_values(heads, kv, dim, cache, dtype, name, pages):
    """One at a first position, at a last one, of either sign, both signs of an element, and a NaN: wherever the
    weight is a power of two, or has a low part of either sign."""
    q, keys, values, table, lengths = _case(LENGTHS[name], heads, kv, dim, 16, dtype, cache, seed=dim)

    def put(b, t, head, e, what):
        values[table[b, t // 16], t % 16, head, e] = what

    for b, n in enumerate(lengths.tolist()):
        if n == 0:
            continue
        put(b, 0, 0, 3, INF), put(b, n - 1, kv - 1, 5, -INF), put(b, n // 2, 0, dim - 1, INF)
        if n > 1:
            put(b, n - 1, 0, 9, INF), put(b, 0, 0, 9, -INF)
        put(b, n // 3, kv - 1, 11, NAN)
        for t in range(0, n, 7):
            put(b, t, 0, 1, INF)
    out = _check(q, keys, values, _wide(table, pages), lengths)
    assert torch.isinf(out).any() and torch.isnan(out).any() and torch.isfinite(out).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [33, 700, 5000])
def test_an_infinite_value_of_small_weight(n, dtype):
    """2^-40 of the largest weight, which float16 has not got."""
    q = torch.full((1, 2, 16), 2.0, dtype=dtype)
    keys = torch.zeros((n, 1, 1, 16), dtype=dtype)
    values = torch.ones((n, 1, 1, 16), dtype=dtype)
    keys[n - 2] = 1.0  # its score: 32 scale
    values[3, 0, 0, 2], values[n // 2, 0, 0, 7] = INF, -INF
    out = _check(q, keys, values, torch.arange(n)[None], torch.tensor([n]), scale=40 * np.log(2.0) / 32)
    assert (out[..., 2] == INF).all() and (out[..., 7] == -INF).all() and out.isinf().sum() == 4


@pytest.mark.parametrize("pages", [0, 1, 30, 1000])
@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (32, 8, 128), (3, 1, 240)])
def test_large_values(heads, kv, dim, dtype, name, pages):
    """1e38 to 3e38: three of them are more than float32 holds."""
    q, keys, values, table, lengths = _case(LENGTHS[name], heads, kv, dim, 16, dtype, seed=dim)
    g = torch.Generator().manual_seed(1)
    values = ((1.0 + 2.0 * torch.rand(values.shape, generator=g)) * 1e38).to(dtype)
    values[..., 1::2] *= -1
    _check(q, keys, values, _wide(table, pages), lengths)


def test_large_and_infinite_values_of_many_sequences():
    """A wave each."""
    g = torch.Generator().manual_seed(2)
    q, keys, values, table, lengths = _case(torch.randint(0, 64, (900,), generator=g).tolist(), 4, 2, 64, 16,
                                            torch.bfloat16, seed=3)
    values[:, 5] = ((1.0 + 2.0 * torch.rand(values[:, 5].shape, generator=g)) * 1e38).to(torch.bfloat16)
    values[::3, 9, :, 4] = INF
    _check(q, keys, values, table, lengths)


@pytest.mark.parametrize("pages", [0, 1000])
def test_the_rest_keeps_its_bits(pages):
    """float16: heads and sequences beside an infinite value, and its own head's other elements."""
    q, keys, values, table, lengths = _case([1200, 5, 333], 8, 2, 64, 16, torch.float16, seed=4)
    args = q.cuda(), keys.cuda()
    rest = _wide(table, pages).cuda(), lengths.cuda()
    want = K.paged_attention(*args, values.cuda(), *rest)
    values[table[0, 10], 3, 0, 7] = INF
    got = K.paged_attention(*args, values.cuda(), *rest)
    assert (got[0, :4, 7] == INF).all()
    got[0, :4, 7] = want[0, :4, 7]
    assert torch.equal(got, want)
