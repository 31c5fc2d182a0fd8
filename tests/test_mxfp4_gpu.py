"""MXFP4 quantisation and its inverse, bit for bit, and the MXFP4 product, against
the float64 restatements in oracle/products.py.

Products: e2m1 products are multiples of 1/4 of at most 36, so with scales within a
factor 2^s of each other every partial sum is a multiple of 2^(-2 - s) below
36 L 2^s of the smallest unit: exact in float32 for small L and s, in any order. Those
are compared bit for bit. Otherwise the float32 sum of L products is off by at most
(L + 2) 2^-24 x sum |a b|, and the result's rounding by eps / 2 x |result|.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from oracle import products

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = [str(d).split(".")[-1] for d in DTYPES]
U = 2.0 ** -24


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bytes(t):
    return t.view(torch.uint8).cpu().numpy()


def _check_quant(x):
    """Codes and scales bit for bit, and the values back."""
    codes, scales = K.mxfp4_quant(x.cuda())
    want_c, want_s = products.mxfp4_quant(x.double().numpy())
    assert codes.dtype == torch.uint8 and scales.dtype == torch.float8_e8m0fnu
    assert codes.shape == want_c.shape and scales.shape == want_s.shape
    assert np.array_equal(_bytes(scales), want_s)
    bad = np.argwhere(_bytes(codes) != want_c)
    assert not len(bad), (bad[:4].tolist(), _bytes(codes)[tuple(bad[0])], want_c[tuple(bad[0])])
    for dtype in DTYPES:
        got = K.mxfp4_dequant(codes, scales, x.shape[-1], dtype).cpu()
        exact = products.mxfp4_values(want_c, want_s, x.shape[-1])
        want = torch.from_numpy(exact).to(dtype)
        assert got.shape == x.shape and got.dtype == dtype
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0)), dtype


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 32), (3, 31), (5, 33), (64, 64), (7, 200), (2, 3, 96), (130, 129), (96,),
                                   (1000, 257), (17, 4096)], ids=lambda s: "x".join(map(str, s)))
def test_quant(shape, dtype):
    x = torch.randn(shape, generator=_gen(sum(shape)))
    _check_quant((x * torch.exp2(torch.randint(-12, 12, (*shape[:-1], 1), generator=_gen(1)).float())).to(dtype))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_every_border(dtype):
    """Values on, next to and between the borders of the codes, of both signs, under a
    block maximum in [4, 8) that makes the scale 1; and scaled by powers of two."""
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 7.0, 0.0])
    eps = torch.finfo(dtype).eps
    near = torch.cat([mid, mid * (1 + eps), mid * (1 - eps), mid * (1 + 3 * eps)])
    v = torch.cat([near, -near])
    blocks = torch.stack([torch.cat([torch.tensor([top]), part]) for top in (4.0, 5.9, 7.9) for part in v.split(31)
                          if len(part) == 31])
    for power in (0, -3, 9):
        _check_quant((blocks * 2.0 ** power).to(dtype))


def test_every_bfloat16():
    """All 65536 bfloat16 values as blocks' largest magnitude, with neighbours of every size: subnormals, the
    clamped scales at 2^-127, infinities and NaNs."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    factors = torch.tensor([1.0, 0.5, 0.75, -0.3, 0.126, -0.9, 0.0, 1e-3])
    x = (bits.float()[:, None] * factors).to(torch.bfloat16)
    _check_quant(x.reshape(-1, 32))  # four values and their neighbours a block
    _check_quant(x)                  # one, in a partial block


def test_float32_extremes():
    tiny, big = 2.0 ** -149, 3.4028234663852886e38
    rows = [[tiny, 0.0, -tiny], [2.0 ** -126, 2.0 ** -127, -(2.0 ** -130)], [2.0 ** -125, 1.9 * 2.0 ** -125, 0.0],
            [big, -big, 1.0], [-0.0, 0.0, -0.0], [float("inf"), 1.0, 2.0], [1.0, float("nan"), 2.0],
            [2.0 ** 127, -(2.0 ** 126), 2.0 ** 125], [float("-inf"), float("nan"), 0.0]]
    x = torch.zeros(len(rows), 70)
    x[:, :3] = torch.tensor(rows, dtype=torch.float64).float()
    x[:, 40:43] = torch.randn(len(rows), 3, generator=_gen(0))  # the next block is not touched by this one's
    _check_quant(x)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("off", [1, 3])
def test_unaligned_rows(off, dtype):
    from tests import _cck

    lib, tag = _cck.load(), DTYPES.index(dtype)
    rows, width = 37, 96
    x = torch.randn(rows * width + 16, generator=_gen(off)).to(dtype)
    want_c, want_s = products.mxfp4_quant(x[off:off + rows * width].reshape(rows, width).double().numpy())
    xd = x.cuda()
    codes = torch.full((rows * 48 + 64,), 9, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows * 3 + 64,), 9, dtype=torch.uint8, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    assert lib.launch_mxfp4_quant_fwd(xd.data_ptr() + off * x.element_size(), codes.data_ptr() + 4,
                                      scales.data_ptr() + off, rows, width, tag, st) == 0
    torch.cuda.synchronize()
    assert np.array_equal(codes[4:4 + rows * 48].cpu().numpy().reshape(rows, 48), want_c)
    assert np.array_equal(scales[off:off + rows * 3].cpu().numpy().reshape(rows, 3), want_s)
    assert (codes[:4] == 9).all() and (codes[4 + rows * 48:] == 9).all()
    assert (scales[:off] == 9).all() and (scales[off + rows * 3:] == 9).all()
    out = torch.full((rows * width + 16,), 5, dtype=dtype, device="cuda")
    assert lib.launch_mxfp4_dequant_fwd(codes.data_ptr() + 4, scales.data_ptr() + off,
                                        out.data_ptr() + off * out.element_size(), rows, width, tag, st) == 0
    torch.cuda.synchronize()
    want = torch.from_numpy(products.mxfp4_values(want_c, want_s, width)).to(dtype)
    assert torch.equal(out[off:off + rows * width].cpu().reshape(rows, width), want)
    assert (out[:off] == 5).all() and (out[off + rows * width:] == 5).all()


def _random_pair(shape, width, seed, low=125, high=129):
    """Random codes (zeros past the width) and scale bytes in [low, high]."""
    blocks = -(-width // 32)
    g = _gen(seed)
    codes = torch.randint(0, 16, (*shape, blocks * 32), generator=g, dtype=torch.uint8)
    codes[..., width:] = 0
    scales = torch.randint(low, high + 1, (*shape, blocks), generator=g, dtype=torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, scales.view(torch.float8_e8m0fnu)


def _values(pair, width):
    return products.mxfp4_values(pair[0].numpy(), pair[1].view(torch.uint8).numpy(), width)


def _check_linear(sizes, n, k, dtype, seed=0, first=0, rows=None, low=125, high=129, dense=False):
    offsets = np.concatenate([[first], first + np.cumsum(sizes)])
    rows = int(offsets[-1]) if rows is None else rows
    x = _random_pair((rows,), k, seed, low, high)
    w = _random_pair((n,) if dense else (len(sizes), n), k, seed + 1, low, high)
    o = None if dense else torch.from_numpy(offsets).cuda()
    got = K.mxfp4_linear(*(t.cuda() for t in (*x, *w)), o, dtype).cpu()
    xv, wv = _values(x, k), _values(w, k)
    if dense:
        wv, offsets = wv[None], np.array([0, rows])
    exact = products.grouped_linear(xv, wv, offsets)
    assert got.dtype == dtype and got.shape == exact.shape
    # units of the smallest product: at most 36 k 4 2^(2 (high - low)) of them in a sum
    if high - low <= 4 and 36 * k * 4 * 2 ** (2 * (high - low)) < 2 ** 24:
        assert torch.equal(got, torch.from_numpy(exact).to(dtype))
        return
    sum_error = (k + 2) * U * products.grouped_linear(np.abs(xv), np.abs(wv), offsets)
    bound = sum_error + torch.finfo(dtype).eps / 2 * (np.abs(exact) + sum_error) + torch.finfo(dtype).tiny
    off = np.abs(got.double().numpy() - exact) > bound
    assert not off.any(), (int(off.sum()), np.argwhere(off)[:3].tolist())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (16, 16, 32), (5, 130, 96), (128, 128, 256), (33, 72, 257),
                                      (130, 260, 520), (3, 1000, 288), (300, 24, 64)])
def test_dense_products(rows, n, k, dtype):
    _check_linear([rows], n, k, dtype, seed=rows + n, dense=True, low=126, high=128)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sizes", [[1], [0, 5, 0], [127, 1, 129], [16, 17, 0, 300], [2] * 65],
                         ids=lambda s: "x".join(map(str, s))[:20])
@pytest.mark.parametrize("k", [128, 320, 90])
def test_grouped_products(sizes, k, dtype):
    _check_linear(sizes, 140, k, dtype, seed=k, low=126, high=128)


def test_rows_of_no_expert_are_zero():
    _check_linear([30, 0, 5], 40, 64, torch.bfloat16, first=3, rows=77, low=127, high=128)


@pytest.mark.parametrize("k", [1024, 4096 + 32])
def test_long_sums_and_distant_scales(k):
    for dtype in DTYPES[::2]:
        _check_linear([40, 3], 70, k, dtype, seed=k, low=107, high=140)


def test_scales_of_nan_reach_their_rows_only():
    x, w = _random_pair((20,), 128, 0), _random_pair((18,), 128, 1)
    xs, ws = x[1].view(torch.uint8), w[1].view(torch.uint8)
    xs[3, 2] = 255
    ws[7, 0] = 255
    got = K.mxfp4_linear(*(t.cuda() for t in (*x, *w))).cpu()
    want = torch.zeros(20, 18, dtype=torch.bool)
    want[3], want[:, 7] = True, True
    assert torch.equal(got.isnan(), want)


def test_quantised_layer():
    """Quantise, multiply and compare with the product of the values, from floats."""
    x, w = torch.randn(70, 200, generator=_gen(5)).bfloat16(), torch.randn(90, 200, generator=_gen(6)).bfloat16()
    xp, wp = K.mxfp4_quant(x.cuda()), K.mxfp4_quant(w.cuda())
    got = K.mxfp4_linear(*xp, *wp, out_dtype=torch.float32).cpu().double().numpy()
    xv, wv = (products.mxfp4_values(*products.mxfp4_quant(t.double().numpy()), 200) for t in (x, w))
    assert (np.abs(got - xv @ wv.T) <= 204 * U * (np.abs(xv) @ np.abs(wv).T)).all()


def test_nothing_to_sum():
    c, s = K.mxfp4_quant(torch.zeros(3, 0, device="cuda"))
    assert c.shape == (3, 0) and s.shape == (3, 0)
    wc, ws = K.mxfp4_quant(torch.zeros(5, 0, device="cuda"))
    assert torch.equal(K.mxfp4_linear(c, s, wc, ws), torch.zeros(3, 5, dtype=torch.bfloat16, device="cuda"))
    c, s = K.mxfp4_quant(torch.zeros(0, 64, device="cuda"))
    wc, ws = K.mxfp4_quant(torch.zeros(5, 64, device="cuda"))
    assert K.mxfp4_linear(c, s, wc, ws).shape == (0, 5)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_launcher_writes_sums_of_nothing(dtype):
    from tests import _cck

    rows, n, st = 300, 70, torch.cuda.current_stream().cuda_stream
    o = torch.tensor([0, 120, 290], device="cuda")
    for offsets, experts in ((None, 1), (o.data_ptr(), 2)):
        out = torch.full((rows * n + 16,), 55, dtype=dtype, device="cuda")
        assert _cck.load().launch_mxfp4_linear_fwd(None, None, None, None, offsets, out.data_ptr(), rows, experts, n, 0,
                                                   DTYPES.index(dtype), st) == 0
        torch.cuda.synchronize()
        assert (out[:rows * n] == 0).all() and (out[rows * n:] == 55).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("k", [128, 256, 384, 640])
def test_large_tiles(k, dtype):
    """Rows and columns enough for the largest tiles, full and cut; odd and even numbers of steps."""
    _check_linear([300, 1, 0, 900, 129], 7442, k, dtype, seed=k, first=3, rows=1500, low=126, high=128)


def test_large_tiles_dense():
    _check_linear([1930], 6656, 512, torch.bfloat16, seed=2, dense=True, low=126, high=128)


@pytest.mark.parametrize("per", [1, 16, 17, 32, 33, 127, 129])
def test_rows_a_group(per):
    """Either side of the average group sizes that other kernels take, with uneven groups."""
    _check_linear([0, 2 * per, per, per + 1, per - 1], 8200, 128, torch.bfloat16, seed=per, low=126, high=128)
    for k in (256, 224):
        _check_linear([per], 150, k, torch.bfloat16, seed=per, dense=True, low=126, high=128)
        _check_linear([0, 2 * per, per, per + 1, per - 1], 150, k, torch.bfloat16, seed=per, low=126, high=128)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,k", [(8200, 90), (8200, 160), (8200, 288), (8203, 32), (8193, 256), (8200, 256), (8200, 384)])
@pytest.mark.parametrize("sizes", [[130, 0, 250, 1, 20], [300, 130, 0, 77, 100]], ids=["small", "large"])
def test_middle_tiles(sizes, n, k, dtype):
    """192 tiles of 128 x 128 and more: whole steps of four blocks, and any number of blocks."""
    _check_linear(sizes, n, k, dtype, seed=k, first=2, rows=sum(sizes) + 42, low=126, high=128)


SCALE_BYTES = [0, 1, 2, 126, 128, 252, 253, 254]


@pytest.mark.parametrize("rows,n", [(8, 8), (16, 8200), (24, 40), (40, 40), (40, 24576), (256, 38400)],
                         ids=["stream16x16", "stream16x32", "stream32x32", "tiles64", "tiles128", "tiles256"])
@pytest.mark.parametrize("k", [32, 96, 128, 384])
def test_scales_of_every_size(rows, n, k):
    """The ends of E8M0, and scales whose product is ordinary where neither is: a row's blocks share a scale, and all
    codes are positive, so a sum grows to its value, which float32 holds, or which is past its range: infinity. A sum
    below the smallest normal number may be off by that (the bound's last term)."""
    g = _gen(rows + k)
    pairs = []
    for count in (rows, n):
        codes = torch.randint(0, 8, (count, -(-k // 32) * 32), generator=g, dtype=torch.uint8)
        scales = torch.tensor(SCALE_BYTES, dtype=torch.uint8)[torch.arange(count) % 8, None].expand(-1, -(-k // 32))
        pairs.append((codes[:, 0::2] | codes[:, 1::2] << 4, scales.contiguous().view(torch.float8_e8m0fnu)))
    got = K.mxfp4_linear(*(t.cuda() for p in pairs for t in p), out_dtype=torch.float32).cpu().double().numpy()
    exact = _values(pairs[0], k) @ _values(pairs[1], k).T
    past = exact >= 2.0 ** 128
    assert (got[past] == np.inf).all() and past.any()
    got, exact = got[~past], exact[~past]
    bound = (k + 2) * U * exact + torch.finfo(torch.float32).tiny
    off = ~(np.abs(got - exact) <= bound)
    assert not off.any(), (int(off.sum()), got[off][:4], exact[off][:4])
