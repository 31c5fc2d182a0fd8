"""fp8_quant in groups of 128, bit for bit, and fp8_block_linear against float64.

Products of FP8 codes are exact in float32. Where codes and scales keep every partial sum
an integer below 2^24, so is the result in any order: compared bit for bit. Otherwise a
block's float32 sum of 128 products is off by at most 128 2^-24 of the sum of their
magnitudes, its scaling by the two scales' product and the sum over B blocks by (B + 3)
2^-24 more: (131 + B) 2^-24 sum |x w| and the result's rounding, eps / 2 of it.

For 16-bit results the matrix instructions take FP8 codes as they are, and sum eight
products at a time with what is below 2^-13 of the largest one's power of two cut off each
(test_what_the_fp8_instructions_cut_off): seven of the eight lose less than 2^-13 of the
largest each. Which eight of a block meet is the kernel's matter, but the largest of a group
is one of its products, so all groups' largest sum up to no more than all products do: 7
2^-13 sum |x w| in all.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import fp8_format as ff
from custom_cuda_kernals_amd import kernels as K
from oracle import decode
from oracle import fp8 as ofp8

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = [str(d).split(".")[-1] for d in DTYPES]
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
NAME = {v: k for k, v in FP8.items()}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _bytes(t):
    return t.view(torch.uint8).cpu().numpy()


# ---------------------------------------------------------------------------
# The quantiser.
# ---------------------------------------------------------------------------

def _check_group(x, fmt):
    codes, scale = K.fp8_quant(x.cuda(), fmt, "group")
    want_c, want_s = decode.quant_group(x.float().numpy(), fmt)
    assert codes.dtype == FP8[fmt] and scale.shape == want_s.shape
    got_s = scale.cpu().numpy()
    nan = np.isnan(want_s)
    assert np.array_equal(np.isnan(got_s), nan)
    assert np.array_equal(got_s[~nan].view(np.uint32), want_s[~nan].view(np.uint32))
    bad = _bytes(codes) != want_c
    quiet = np.isnan(ofp8.decode(want_c, fmt)) & np.isnan(ofp8.decode(_bytes(codes), fmt))  # a NaN's sign is free
    assert not (bad & ~quiet).any(), np.argwhere(bad & ~quiet)[:4]


@pytest.mark.parametrize("fmt", FP8)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 1), (1, 127), (1, 128), (3, 129), (5, 255), (2, 7), (64, 4096), (333, 777),
                                   (17, 1030), (1000, 384), (70000, 9), (4, 14336)], ids=lambda s: f"{s[0]}x{s[1]}")
def test_group(shape, dtype, fmt):
    x = torch.randn(shape, generator=_gen(sum(shape)))
    far = torch.rand(shape, generator=_gen(1)) < 0.01
    x = torch.where(far, x * 50.0, x) * torch.exp2(torch.randint(-6, 6, (shape[0], 1), generator=_gen(2)).float())
    _check_group(x.to(dtype), fmt)


@pytest.mark.parametrize("fmt", FP8)
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_group_special_values(dtype, fmt):
    x = torch.randn((8, 300), generator=_gen(3)).to(dtype)
    x[0, 5], x[1, 200], x[2, 299], x[3] = float("nan"), float("inf"), -float("inf"), 0.0
    x[4], x[5, :128] = torch.finfo(dtype).tiny / 4, torch.finfo(dtype).max
    x[6, 128:256] = -0.0
    _check_group(x, fmt)


def test_group_unaligned_and_dequantized():
    flat = torch.randn(9 * 256 + 1, generator=_gen(4)).to(torch.bfloat16).cuda()
    x = flat[1:].view(9, 256)
    codes, scale = K.fp8_quant(x, "e4m3", "group")
    again, scale2 = K.fp8_quant(x.clone(), "e4m3", "group")
    assert torch.equal(codes.view(torch.uint8), again.view(torch.uint8)) and torch.equal(scale, scale2)
    ff.check_pair(codes, scale, "group")
    want = decode.block_values(_bytes(codes), scale.cpu().numpy(), "e4m3", False).astype(np.float32)
    assert np.array_equal(ff.dequantize(codes, scale, "group").cpu().numpy(), want)
    x = torch.empty(0, 256, device="cuda")
    assert K.fp8_quant(x, "e4m3", "group")[1].shape == (0, 2)
    assert K.fp8_quant(x.t(), "e4m3", "group")[1].shape == (256, 0)


# ---------------------------------------------------------------------------
# The product.
# ---------------------------------------------------------------------------

def _random(rows, n, k, experts, fx, fw, tall, seed):
    g = _gen(seed)
    shape = (n, k) if experts is None else (experts, n, k)
    x, w = torch.randn((rows, k), generator=g), torch.randn(shape, generator=g)
    codes_x, codes_w = x.to(FP8[fx]), w.to(FP8[fw])
    xs = torch.rand((-(-rows // 128) if tall else rows, -(-k // 128)), generator=g) + 0.1
    ws = torch.rand((*shape[:-2], -(-n // 128), -(-k // 128)), generator=g) * 0.02 + 0.001
    return codes_x, xs, codes_w, ws


def _check(x, xs, w, ws, offsets=None, out=torch.bfloat16, tall=False, got=None):
    if got is None:
        got = K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None if offsets is None else offsets.cuda(),
                                 out)
    xv = decode.block_values(_bytes(x), xs.numpy(), NAME[x.dtype], tall)
    wv = decode.block_values(_bytes(w), ws.numpy(), NAME[w.dtype], True)
    rows, n = x.shape[0], w.shape[-2]
    want, size = np.zeros((rows, n)), np.zeros((rows, n))
    spans = [(0, rows, wv)] if offsets is None else [(int(a), int(b), m) for a, b, m in zip(offsets, offsets[1:], wv)]
    for a, b, m in spans:
        want[a:b], size[a:b] = xv[a:b] @ m.T, np.abs(xv[a:b]) @ np.abs(m).T
    info = torch.finfo(out)
    cut = 0.0 if out == torch.float32 else 7 * 2.0 ** -13
    bound = ((131 + xs.shape[-1]) * 2.0 ** -24 + cut) * size + np.maximum(np.abs(want) * info.eps / 2,
                                                                   info.smallest_normal * info.eps / 2)
    off = np.abs(got.double().cpu().numpy() - want)
    assert got.dtype == out and got.shape == want.shape
    assert (off <= bound).all(), (off / np.maximum(bound, 1e-300)).max()
    return got


@pytest.mark.parametrize("fx,fw", [("e4m3", "e4m3"), ("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("tall", [False, True], ids=["group", "block"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 16, 16), (3, 5, 15), (8, 256, 512), (16, 300, 384), (17, 130, 129),
                                      (33, 65, 1030), (100, 200, 272), (129, 129, 128), (300, 700, 144)])
def test_dense(rows, n, k, tall, fx, fw):
    _check(*_random(rows, n, k, None, fx, fw, tall, rows + n + k), tall=tall)


@pytest.mark.parametrize("out", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,n,k", [(5, 77, 256), (20, 8200, 640), (700, 3000, 256), (2600, 4100, 160), (4096, 2816, 400),
                                      (200, 500, 333), (2000, 2000, 77)])
def test_dense_output_types_and_tiles(rows, n, k, out):
    _check(*_random(rows, n, k, None, "e4m3", "e4m3", False, rows), out=out)


OFFSETS = {
    "few": [0, 1, 1, 3, 4, 4, 9],
    "gaps": [5, 5, 40, 170, 171, 300, 431],
    "large": [0, 700, 700, 901, 1400, 1401, 2000],
}


@pytest.mark.parametrize("tall", [False, True], ids=["group", "block"])
@pytest.mark.parametrize("n,k", [(200, 256), (1412, 1030), (2304, 384)])
@pytest.mark.parametrize("name", OFFSETS)
def test_grouped(name, n, k, tall):
    offsets = torch.tensor(OFFSETS[name])
    rows = int(offsets[-1]) + 7
    got = _check(*_random(rows, n, k, 6, "e4m3", "e4m3", tall, n), offsets=offsets, out=torch.float32, tall=tall)
    assert (got[:int(offsets[0])] == 0).all() and (got[int(offsets[-1]):] == 0).all()


def test_grouped_in_no_order():
    """Offsets in no order, or past the rows: some result, and no row outside."""
    x, xs, w, ws = _random(300, 200, 256, 4, "e4m3", "e4m3", False, 9)
    for offsets in ([300, 200, 100, 50, 0], [0, 250, 10, 400, 300], [-9, 1 << 40, 5, -3, 200], [0, 0, 0, 0, 0]):
        for rows in (2, 40, 300):
            y = K.fp8_block_linear(x[:rows].cuda(), xs[:rows].cuda(), w.cuda(), ws.cuda(),
                                   torch.tensor(offsets).cuda(), torch.float32)
            assert y.shape == (rows, 200)


def _whole(shape, seed, fmt):
    """Integers -4 .. 4."""
    return torch.randint(-4, 5, shape, generator=_gen(seed)).float().to(FP8[fmt])


@pytest.mark.parametrize("rows,n,k", [(1, 40, 4096), (7, 513, 2048), (30, 256, 1024), (150, 260, 1040), (257, 1100, 1024),
                                      (3000, 3500, 272), (900, 1100, 1001)])
def test_exact(rows, n, k):
    """Sums of integers times powers of two: below 2^24 of their unit, so equal whatever the order."""
    x, w = _whole((rows, k), 1, "e4m3"), _whole((n, k), 2, "e5m2")
    xs = torch.exp2(torch.randint(-1, 2, (rows, -(-k // 128)), generator=_gen(3)).float())
    ws = torch.exp2(torch.randint(-1, 2, (-(-n // 128), -(-k // 128)), generator=_gen(4)).float())
    got = K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None, torch.float32).cpu().numpy()
    want = (decode.block_values(_bytes(x), xs.numpy(), "e4m3", False)
            @ decode.block_values(_bytes(w), ws.numpy(), "e5m2", True).T)
    assert np.array_equal(got, want)


def test_what_the_fp8_instructions_cut_off():
    """One product of 1 and one of 2^-n, wherever they meet: a 16-bit result is off by less than 2^-13, and by
    nothing for n up to 13 (but for its own rounding: the difference to 1 is what is left of it); float32 has both."""
    k, n = 128, torch.arange(1, 21)
    x = torch.zeros(20, k)
    x[:, 0], x[torch.arange(20), 1 + 6 * torch.arange(20)] = 1.0, torch.exp2(-(n // 2).float())
    w = torch.zeros(20, k)
    w[:, 0] = 1.0
    w[torch.arange(20), 1 + 6 * torch.arange(20)] = torch.exp2(-(n - n // 2).float())
    x, w = x.to(torch.float8_e5m2), w.to(torch.float8_e5m2)
    args = x.cuda(), torch.ones(20, 1).cuda(), w.cuda(), torch.ones(1, 1).cuda(), None
    exact = torch.diagonal(K.fp8_block_linear(*args, torch.float32).cpu())
    assert torch.equal(exact, 1.0 + torch.exp2(-n.float()))
    cut = torch.diagonal(K.fp8_block_linear(*args, torch.float16).cpu()).double()
    off = (cut - exact.double()).abs()
    assert (off <= 2.0 ** -13 + 2.0 ** -11).all()


def test_subnormal_codes_and_extreme_scales():
    x, w = (torch.full((20, 256), v).to(torch.float8_e4m3fn) for v in (2.0 ** -9, 448.0))
    one = torch.ones(20, 2)
    y = K.fp8_block_linear(x.cuda(), one.cuda(), w.cuda(), torch.ones(1, 2).cuda(), None, torch.float32)
    assert (y == 256 * 448.0 * 2.0 ** -9).all()
    y = K.fp8_block_linear(x.cuda(), (one * 1e-30).cuda(), w.cuda(), torch.full((1, 2), 1e30).cuda(), None, torch.float32)
    assert ((y / (256 * 448.0 * 2.0 ** -9) - 1).abs() < 1e-6).all()


@pytest.mark.parametrize("rows,n", [(3, 70), (20, 300), (150, 300), (3000, 3300)])
def test_infinities_and_nan_stay_in_their_rows(rows, n):
    x, xs, w, ws = _random(rows, n, 400, None, "e5m2", "e4m3", False, 12)
    x[rows // 2, 131], x[0, 399] = float("inf"), float("nan")
    y = K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None, torch.float32)
    bad = ~y.isfinite()
    assert bad[0].all() and bad[rows // 2].all() and not bad[1:rows // 2].any() and not bad[rows // 2 + 1:].any()
    x, xs, w, ws = _random(rows, n, 400, None, "e4m3", "e4m3", False, 13)
    w[n // 3, 17] = float("nan")
    bad = ~K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None, torch.float32).isfinite()
    assert bad[:, n // 3].all() and bad.sum() == rows


def test_unaligned_codes():
    for k in (256, 130):
        x, xs, w, ws = _random(40, 90, k, None, "e4m3", "e4m3", False, 14)
        flat = torch.zeros(40 * k + 1, dtype=torch.float8_e4m3fn, device="cuda")
        flat.view(torch.uint8)[1:] = x.view(torch.uint8).flatten().cuda()
        args = xs.cuda(), w.cuda(), ws.cuda(), None, torch.float32
        # another kernel, whose sums may be of another order
        _check(x, xs, w, ws, out=torch.float32, got=K.fp8_block_linear(flat[1:].view(40, k), *args))


def test_nothing():
    e4 = torch.float8_e4m3fn
    x, w = torch.empty(0, 256, device="cuda").to(e4), torch.empty(9, 256, device="cuda").to(e4)
    y = K.fp8_block_linear(x, torch.empty(0, 2, device="cuda"), w, torch.ones(1, 2, device="cuda"))
    assert y.shape == (0, 9)
    y = K.fp8_block_linear(torch.empty(5, 0, device="cuda").to(e4), torch.empty(5, 0, device="cuda"),
                           torch.empty(9, 0, device="cuda").to(e4), torch.empty(1, 0, device="cuda"))
    assert y.shape == (5, 9) and (y == 0).all()


def test_rows_behind_and_before_stay():
    """A product into part of a larger tensor's memory leaves the rest."""
    from custom_cuda_kernals_amd._lib import native

    for rows, n, k in ((3, 300, 256), (100, 130, 250), (2600, 4100, 160)):
        x, xs, w, ws = _random(rows, n, k, None, "e4m3", "e4m3", False, 15)
        room = torch.full((rows + 2, n), 7.0, dtype=torch.bfloat16, device="cuda")
        native.fp8_block_linear_fwd(x.cuda(), xs.cuda(), w.cuda(), ws.cuda(), None, room[1:-1])
        _check(x, xs, w, ws, got=room[1:-1])
        assert (room[0] == 7).all() and (room[-1] == 7).all()


def test_gradients_are_the_same_operator_on_transposed_tiles():
    """Of the loss sum(y * g) with every operand in 128 x 128 tiles: the formula's, from the codes' values."""
    rows, n, k = 300, 200, 260
    x, w, g = (torch.randn(s, generator=_gen(20 + i)).to(torch.bfloat16)
               for i, s in enumerate(((rows, k), (n, k), (rows, n))))
    (xc, xs), (wc, ws), (gc, gs) = ((t for t in K.fp8_quant(a.cuda(), f, "block"))
                                    for a, f in ((x, "e4m3"), (w, "e4m3"), (g, "e5m2")))
    grad_x = K.fp8_block_linear(gc, gs, wc.t().contiguous(), ws.t().contiguous(), None, torch.float32)
    grad_w = K.fp8_block_linear(gc.t().contiguous(), gs.t().contiguous(), xc.t().contiguous(), xs.t().contiguous(), None,
                                torch.float32)
    xv, wv, gv = (torch.from_numpy(decode.block_values(_bytes(c), s.cpu().numpy(), f, True))
                  for c, s, f in ((xc, xs, "e4m3"), (wc, ws, "e4m3"), (gc, gs, "e5m2")))
    a, b = xv.clone().requires_grad_(), wv.clone().requires_grad_()
    ((a @ b.t()) * gv).sum().backward()
    for got, want, size in ((grad_x, a.grad, gv.abs() @ wv.abs()), (grad_w, b.grad, gv.abs().t() @ xv.abs())):
        assert ((got.double().cpu() - want).abs() <= 140 * 2.0 ** -24 * size + want.abs() * 2.0 ** -24).all()


def test_same_bits_every_time():
    for rows in (5, 25, 200, 3000):
        args = [t.cuda() for t in _random(rows, 3000, 512, None, "e4m3", "e4m3", False, 30)]
        first = K.fp8_block_linear(*args)
        assert all(torch.equal(K.fp8_block_linear(*args), first) for _ in range(3))


@pytest.mark.parametrize("out", [torch.float16, torch.bfloat16], ids=IDS[1:])
@pytest.mark.parametrize("tall", [False, True], ids=["group", "block"])
@pytest.mark.parametrize("rows,n,k", [(4100, 3700, 272), (2100, 8200, 2064), (4352, 3590, 128)])
def test_large_tiles(rows, n, k, tall, out):
    _check(*_random(rows, n, k, None, "e5m2", "e4m3", tall, k), out=out, tall=tall)


def test_large_tiles_of_groups():
    offsets = torch.tensor([3, 1000, 1000, 2100, 3001, 3002, 4400])
    got = _check(*_random(4407, 3700, 400, 6, "e4m3", "e5m2", False, 40), offsets=offsets)
    assert (got[:3] == 0).all() and (got[4400:] == 0).all()


@pytest.mark.parametrize("rows,n", [(3, 70), (20, 300), (150, 300), (3000, 3300), (4100, 3700)])
def test_infinities_and_nan_of_16_bit_results(rows, n):
    x, xs, w, ws = _random(rows, n, 400, None, "e5m2", "e4m3", False, 41)
    x[rows // 2, 131], x[0, 399] = float("inf"), float("nan")
    w[n // 3, 17] = float("nan")
    bad = ~K.fp8_block_linear(x.cuda(), xs.cuda(), w.cuda(), ws.cuda()).isfinite()
    assert bad[0].all() and bad[rows // 2].all() and bad[:, n // 3].all()
    assert bad.sum() == 2 * n + rows - 2
