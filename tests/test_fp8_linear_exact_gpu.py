"""fp8_block_linear with 16-bit results, bit for bit.

The FP8 instructions sum eight neighbouring products with the bits below 2^-13 of the
largest one's power of two cut off. Products of the integers -4 .. 4 are 16 at most, so
nothing of them is cut off; a block's sum is an integer of 2^11 at most, times its scales,
powers of two, and all blocks' sum is exact in float32. The result is that sum, rounded
once: one lost or misplaced code is seen. The kernels, by size: streams of 16 and 32 rows,
tiles of 64, 128 and 256, rows that are no whole vectors, and rows of fewer than 16 codes.

What is cut off shows by cancellation: products 1 and 2^-n in one block, -1 in the next.
Those two are then 2^-n if it was kept and 0 if not, both exact in float16.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from oracle import decode
from tests.test_fp8_linear_gpu import FP8, _bytes, _gen, _whole

pytestmark = pytest.mark.gpu

HALF = [torch.float16, torch.bfloat16]
IDS = ["float16", "bfloat16"]


def _scales(shape, seed):
    return torch.exp2(torch.randint(-1, 2, shape, generator=_gen(seed)).float())


def _operands(rows, n, k, experts, tall, fx, fw):
    x, w = _whole((rows, k), rows, fx), _whole((n, k) if experts is None else (experts, n, k), n, fw)
    xs = _scales((-(-rows // 128) if tall else rows, -(-k // 128)), 3)
    ws = _scales((*w.shape[:-2], -(-n // 128), -(-k // 128)), 4)
    return x, xs, w, ws


def _rounded(want, out):
    assert np.array_equal(want.astype(np.float32), want)  # exact so far
    return torch.from_numpy(want.astype(np.float32)).to(out)


def _values(x, xs, w, ws, tall, fx, fw):
    return decode.block_values(_bytes(x), xs.numpy(), fx, tall), decode.block_values(_bytes(w), ws.numpy(), fw, True)


SIZES = [(1, 40, 4096), (7, 513, 2048), (16, 14336, 512), (24, 700, 1024), (30, 256, 1040), (150, 260, 1040),
         (200, 1100, 2064), (700, 2900, 272), (2600, 4100, 160), (4100, 3700, 272), (2100, 8200, 2064), (900, 1100, 1001),
         (3, 77, 4095), (300, 200, 15)]


@pytest.mark.parametrize("out", HALF, ids=IDS)
@pytest.mark.parametrize("tall", [False, True], ids=["group", "block"])
@pytest.mark.parametrize("rows,n,k", SIZES)
def test_dense(rows, n, k, tall, out):
    x, xs, w, ws = _operands(rows, n, k, None, tall, "e4m3", "e5m2")
    got = K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None, out).cpu()
    a, b = _values(x, xs, w, ws, tall, "e4m3", "e5m2")
    assert torch.equal(got, _rounded(a @ b.T, out))


@pytest.mark.parametrize("out", HALF, ids=IDS)
@pytest.mark.parametrize("offsets", [[0, 1, 1, 3, 4, 4, 9], [5, 5, 40, 170, 171, 300, 431], [0, 700, 700, 901, 1400, 1401, 2000],
                                     [3, 1000, 1000, 2100, 3001, 3002, 4400]], ids=["few", "gaps", "large", "tiles"])
@pytest.mark.parametrize("n,k", [(200, 256), (1412, 1030), (3700, 400)])
def test_grouped(n, k, offsets, out):
    rows = offsets[-1] + 7
    x, xs, w, ws = _operands(rows, n, k, 6, False, "e5m2", "e4m3")
    got = K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), torch.tensor(offsets).cuda(), out).cpu()
    a, b = _values(x, xs, w, ws, False, "e5m2", "e4m3")
    want = np.zeros((rows, n))
    for first, last, m in zip(offsets, offsets[1:], b):
        want[first:last] = a[first:last] @ m.T
    assert torch.equal(got, _rounded(want, out))


@pytest.mark.parametrize("fx,fw", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("rows,n", [(9, 300), (30, 300), (200, 300), (2600, 4100), (4100, 3700)])
def test_formats(rows, n, fx, fw):
    x, xs, w, ws = _operands(rows, n, 384, None, False, fx, fw)
    got = K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None, torch.bfloat16).cpu()
    a, b = _values(x, xs, w, ws, False, fx, fw)
    assert torch.equal(got, _rounded(a @ b.T, torch.bfloat16))


@pytest.mark.parametrize("wide", [1, 30], ids=["128", "3840"])
@pytest.mark.parametrize("times", [1, 2, 20, 256], ids=["16 rows", "32 rows", "320 rows", "4096 rows"])
@pytest.mark.parametrize("first", [0, 5, 63, 127])
def test_what_the_fp8_instructions_cut_off(first, times, wide):
    """Product 1 at place `first` and 2^-n at every other place of a block, a column each, 1 <= n <= 16: kept down to
    2^-13 wherever the two meet, and below it cut off, or kept where they meet in float32; a float32 result has all."""
    n = torch.arange(1, 17)
    x = torch.exp2(-n.float())[:, None].repeat(1, 256)
    x[:, 128:] = 0.0
    x[:, first], x[:, 128] = 1.0, -1.0
    w = torch.eye(128, 256)
    w[:, first] = w[:, 128] = 1.0
    w[first] = 0.0
    x, w = x.repeat(times, 1).to(FP8["e5m2"]), w.repeat(wide, 1).to(FP8["e5m2"])
    args = x.cuda(), torch.ones(16 * times, 2).cuda(), w.cuda(), torch.ones(wide, 2).cuda(), None
    want = torch.exp2(-n.double())[:, None].repeat(times, 128 * wide)
    want[:, first::128] = 0.0
    assert torch.equal(K.fp8_block_linear(*args, torch.float32).cpu().double(), want)
    for out in HALF:
        got = K.fp8_block_linear(*args, out).cpu().double()
        assert ((got == want) | (got == 0.0)).all()
        kept = n.repeat(times) <= 13
        assert torch.equal(got[kept], want[kept])
        lost = (got[~kept] == 0.0) & (want[~kept] != 0.0)
        # seven neighbours of the eight lose theirs, n 14 to 16, and all copies alike
        assert int(lost.sum()) == 7 * 3 * times * wide, int(lost.sum())
