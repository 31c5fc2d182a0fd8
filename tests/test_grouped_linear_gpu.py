"""grouped_linear and its two gradients against float64 products of each expert's
rows (oracle/products.py).

Two kinds of inputs. Small integers: every product and every partial sum is an
integer below 2^24, so the float32 sums are exact in any order and the result is
the exact sum rounded once to the storage type, bit for bit. Normal values, where
with u = 2^-24 the float32 sum of L products is off by at most
(L + 1) u / (1 - (L + 1) u) x sum |a b| (each product and each sum rounded once, any
order), taken as (L + 2) u x sum |a b|, and the rounding to the storage type by
half a step: eps / 2 x |result| (both terms).
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


def _ints(shape, most, dtype, seed):
    return torch.randint(-most, most + 1, shape, generator=_gen(seed)).to(dtype)


def _normal(shape, dtype, seed):
    return torch.randn(shape, generator=_gen(seed)).to(dtype)


def _offsets(sizes, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(sizes)]), dtype=torch.int64)


def _np(t):
    return t.double().cpu().numpy()


def _rounded(exact, dtype):
    """float64 -> dtype, once (float32 and the 16-bit types round from float64 directly)."""
    return torch.from_numpy(exact).to(dtype)


def _close(got, exact, magnitude, length, dtype, what):
    """|got - exact| within the bounds of the module docstring."""
    g = _np(got)
    sum_error = (length + 2) * U * magnitude
    bound = sum_error + torch.finfo(dtype).eps / 2 * (np.abs(exact) + sum_error) + torch.finfo(dtype).tiny
    off = np.abs(g - exact) > bound
    assert not off.any(), (what, int(off.sum()), np.argwhere(off)[:3].tolist(), g[off][:3], exact[off][:3])


def _three(x, w, g, offsets):
    """All three operators on the GPU: (y, grad_x, grad_w)."""
    x, w, g, o = x.cuda(), w.cuda(), g.cuda(), offsets.cuda()
    return K.grouped_linear(x, w, o), K.grouped_linear_grad_input(g, w, o), K.grouped_linear_grad_weight(g, x, o)


def _exact(x, w, g, offsets):
    x, w, g, o = _np(x), _np(w), _np(g), offsets.numpy()
    return (products.grouped_linear(x, w, o), products.grouped_linear_grad_input(g, w, o),
            products.grouped_linear_grad_weight(g, x, o))


def _check_ints(sizes, n, k, dtype, seed=0, rows=None, first=0):
    offsets = _offsets(sizes, first)
    rows = int(offsets[-1]) if rows is None else rows
    # |sum| <= length x most^2 < 2^24
    most = 4 if max(n, k, rows) < 500_000 else 1
    x, w = _ints((rows, k), most, dtype, seed), _ints((len(sizes), n, k), most, dtype, seed + 1)
    g = _ints((rows, n), most, dtype, seed + 2)
    for got, exact, what in zip(_three(x, w, g, offsets), _exact(x, w, g, offsets), ("y", "grad_x", "grad_w")):
        want = _rounded(exact, dtype)
        assert torch.equal(got.cpu(), want), (what, (got.cpu() != want).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,k", [(1, 1), (8, 8), (16, 128), (128, 64), (130, 72), (264, 200), (65, 33), (7, 300),
                                 (257, 129)])
def test_widths(n, k, dtype):
    """Below, at and past a tile and a step; whole vectors and odd widths."""
    _check_ints([5, 0, 130, 1, 64], n, k, dtype, seed=n + k)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sizes", [[1], [0, 1], [0, 0, 0], [127, 128, 129], [16, 15, 17, 1], [256, 257], [1] * 70,
                                   [0, 300, 0, 0, 1, 0]], ids=lambda s: "x".join(map(str, s))[:20])
def test_group_sizes(sizes, dtype):
    _check_ints(sizes, 72, 96, dtype, seed=len(sizes))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_of_no_expert_are_zero(dtype):
    """Rows before the first group and behind the last: zeros in y and grad_x, and no part of grad_w."""
    _check_ints([3, 40, 0, 7], 48, 56, dtype, rows=90, first=11)
    _check_ints([0, 0], 48, 56, dtype, rows=20, first=20)
    _check_ints([300, 200], 130, 136, dtype, rows=900, first=130)


@pytest.mark.parametrize("experts", [1, 2, 255, 256, 257, 1024])
def test_numbers_of_experts(experts):
    sizes = np.random.default_rng(experts).integers(0, 4, experts).tolist()
    _check_ints(sizes, 24, 40, torch.bfloat16, seed=experts)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,k,rows", [(200, 1000, 300), (96, 2100, 17), (1030, 515, 260)])
def test_normal_values(n, k, rows, dtype):
    sizes = [rows // 2, 0, rows - rows // 2 - 1, 1]
    offsets = _offsets(sizes)
    x, w, g = _normal((rows, k), dtype, 1), _normal((4, n, k), dtype, 2), _normal((rows, n), dtype, 3)
    magnitudes = _exact(x.abs(), w.abs(), g.abs(), offsets)
    for got, exact, mag, length, what in zip(_three(x, w, g, offsets), _exact(x, w, g, offsets), magnitudes,
                                             (k, n, max(sizes)), ("y", "grad_x", "grad_w")):
        _close(got, exact, mag, length, dtype, what)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("off", [1, 2, 4])
def test_unaligned_buffers(off, dtype):
    """Inputs and outputs that begin between two 16-byte vectors, through the C launchers."""
    from tests import _cck

    lib, tag = _cck.load(), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    sizes, n, k = [20, 0, 150], 64, 128
    offsets = _offsets(sizes)
    rows = int(offsets[-1])
    x, w, g = (_ints(s, 4, dtype, i) for i, s in enumerate([(rows, k), (3, n, k), (rows, n)]))

    def moved(t):
        b = torch.full((t.numel() + 16,), 77, dtype=dtype, device="cuda")
        b[off:off + t.numel()] = t.reshape(-1).cuda()
        return b, b.data_ptr() + off * b.element_size()

    o, st = offsets.cuda(), torch.cuda.current_stream().cuda_stream
    xb, wb, gb = moved(x), moved(w), moved(g)
    exact = _exact(x, w, g, offsets)
    for shift in (0, off):
        for what, (fn, a, b) in enumerate([(lib.launch_grouped_linear_fwd, xb, wb),
                                           (lib.launch_grouped_linear_grad_input, gb, wb),
                                           (lib.launch_grouped_linear_grad_weight, gb, xb)]):
            want = _rounded(exact[what], dtype)
            out = torch.full((want.numel() + 16,), 55, dtype=dtype, device="cuda")
            assert fn(a[1], b[1], o.data_ptr(), out.data_ptr() + shift * out.element_size(), rows, 3, n, k, tag, st) == 0
            torch.cuda.synchronize()
            assert torch.equal(out[shift:shift + want.numel()].cpu(), want.reshape(-1)), (what, shift)
            rest = torch.cat([out[:shift], out[shift + want.numel():]])
            assert (rest == 55).all(), "wrote outside the output"


def test_nothing_to_sum():
    o = torch.tensor([0, 2, 5], device="cuda")
    x = torch.zeros(5, 0, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, 8, 0, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(K.grouped_linear(x, w, o), torch.zeros(5, 8, dtype=torch.bfloat16, device="cuda"))
    g = torch.zeros(5, 0, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2, 0, 8, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(K.grouped_linear_grad_input(g, w, o), torch.zeros(5, 8, dtype=torch.bfloat16, device="cuda"))
    none = torch.zeros(3, dtype=torch.int64, device="cuda")
    g, x = (torch.zeros(0, c, dtype=torch.bfloat16, device="cuda") for c in (8, 16))
    w = torch.ones(2, 8, 16, dtype=torch.bfloat16, device="cuda")
    assert K.grouped_linear(x, w, none).shape == (0, 8)
    assert K.grouped_linear_grad_input(g, w, none).shape == (0, 16)
    assert torch.equal(K.grouped_linear_grad_weight(g, x, none), torch.zeros_like(w))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_launchers_write_sums_of_nothing(dtype):
    """Through the C launchers, at any element; nothing around the output."""
    from tests import _cck

    lib, tag = _cck.load(), DTYPES.index(dtype)
    rows, cols, st = 300, 70, torch.cuda.current_stream().cuda_stream
    o = torch.tensor([0, 120, 290], device="cuda")
    for n, k, fn in ((cols, 0, lib.launch_grouped_linear_fwd), (0, cols, lib.launch_grouped_linear_grad_input)):
        out = torch.full((rows * cols + 16,), 55, dtype=dtype, device="cuda")
        assert fn(None, None, o.data_ptr(), out.data_ptr() + out.element_size(), rows, 2, n, k, tag, st) == 0
        torch.cuda.synchronize()
        assert (out[1:1 + rows * cols] == 0).all() and out[0] == 55 and (out[1 + rows * cols:] == 55).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_infinities_and_nan_stay_in_their_rows(dtype):
    """A NaN or infinity in one row, one expert or one column reaches what it is multiplied with, and nothing else;
    rows of no expert are zeros whatever they hold."""
    sizes, n, k = [40, 100, 3], 136, 72
    offsets = _offsets(sizes, 5)
    rows = int(offsets[-1]) + 9
    x, w, g = (_ints(s, 4, dtype, i) for i, s in enumerate([(rows, k), (3, n, k), (rows, n)]))
    x[7, 3], x[60, 71], x[2, 0], x[-1, 5] = float("nan"), float("inf"), float("nan"), float("inf")
    w[2, 9, 1] = float("nan")
    g[50, 0], g[rows - 2, 4] = float("inf"), float("nan")
    for got, exact, what in zip(_three(x, w, g, offsets), _exact(x, w, g, offsets), ("y", "grad_x", "grad_w")):
        want = _rounded(exact, dtype)
        assert torch.equal(got.isnan().cpu(), want.isnan()), what
        assert torch.equal(got.nan_to_num(nan=0.0).cpu(), want.nan_to_num(nan=0.0)), what


@pytest.mark.parametrize("offsets", [[5, 3, 8, 2], [-4, 2, 100, 50], [1 << 40, -(1 << 40), 7, 7], [0, 64, 0, 64]],
                         ids=str)
def test_bad_offsets_touch_nothing_else(offsets):
    """Offsets that decrease or leave the rows: the results are unspecified, but nothing outside the outputs is
    written (the outputs here lie inside larger buffers), and the calls end."""
    from tests import _cck

    lib = _cck.load()
    rows, n, k, pad = 64, 40, 48, 4096
    o = torch.tensor(offsets, device="cuda")
    x, w, g = (torch.ones(s, dtype=torch.bfloat16, device="cuda") for s in [(rows, k), (3, n, k), (rows, n)])
    st = torch.cuda.current_stream().cuda_stream
    for fn, a, b, size in [(lib.launch_grouped_linear_fwd, x, w, rows * n),
                           (lib.launch_grouped_linear_grad_input, g, w, rows * k),
                           (lib.launch_grouped_linear_grad_weight, g, x, 3 * n * k)]:
        out = torch.full((size + 2 * pad,), 55, dtype=torch.bfloat16, device="cuda")
        assert fn(a.data_ptr(), b.data_ptr(), o.data_ptr(), out.data_ptr() + 2 * pad, rows, 3, n, k, 2, st) == 0
        torch.cuda.synchronize()
        assert (out[:pad] == 55).all() and (out[pad + size:] == 55).all()


def test_gradients_against_differences():
    """Central differences of the float32 forward in integers: the layer is linear in each argument, so
    (f(a + 1) - f(a - 1)) / 2 is its derivative exactly."""
    sizes, n, k = [4, 0, 9], 12, 20
    offsets = _offsets(sizes)
    rows = 13
    x, w, g = (_ints(s, 3, torch.float32, i) for i, s in enumerate([(rows, k), (3, n, k), (rows, n)]))
    _, grad_x, grad_w = _three(x, w, g, offsets)
    o = offsets.cuda()

    def loss(x_, w_):
        return float((K.grouped_linear(x_.cuda(), w_.cuda(), o).cpu().double() * g.double()).sum())

    for r, c in [(0, 0), (3, 19), (4, 7), (12, 11)]:
        a, b = x.clone(), x.clone()
        a[r, c] += 1
        b[r, c] -= 1
        assert (loss(a, w) - loss(b, w)) / 2 == float(grad_x[r, c])
    for e, r, c in [(0, 0, 0), (0, 11, 19), (1, 3, 3), (2, 5, 8)]:
        a, b = w.clone(), w.clone()
        a[e, r, c] += 1
        b[e, r, c] -= 1
        assert (loss(x, a) - loss(x, b)) / 2 == float(grad_w[e, r, c])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS[1:])
@pytest.mark.parametrize("k", [8, 64, 72, 136, 200, 264])
def test_large_tiles_forward(k, dtype):
    """Rows and columns enough for the largest tiles: full, cut in rows and in columns at every part of one; from one
    step of the contracted index to five, odd and even."""
    sizes, n = [700, 129, 0, 1, 1100, 641, 40], 7440
    offsets = _offsets(sizes, 3)
    rows = int(offsets[-1]) + 30
    x, w = _ints((rows, k), 4, dtype, k), _ints((len(sizes), n, k), 4, dtype, k + 1)
    got = K.grouped_linear(x.cuda(), w.cuda(), offsets.cuda()).cpu()
    want = _rounded(products.grouped_linear(_np(x), _np(w), offsets.numpy()), dtype)
    assert torch.equal(got, want), (got != want).nonzero()[:4].tolist()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS[1:])
@pytest.mark.parametrize("n", [8, 64, 72, 136, 200, 264])
def test_large_tiles_grad_input(n, dtype):
    sizes, k = [700, 129, 0, 1, 1100, 641, 40], 7440
    offsets = _offsets(sizes, 3)
    rows = int(offsets[-1]) + 30
    g, w = _ints((rows, n), 4, dtype, n), _ints((len(sizes), n, k), 4, dtype, n + 1)
    got = K.grouped_linear_grad_input(g.cuda(), w.cuda(), offsets.cuda()).cpu()
    want = _rounded(products.grouped_linear_grad_input(_np(g), _np(w), offsets.numpy()), dtype)
    assert torch.equal(got, want), (got != want).nonzero()[:4].tolist()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=IDS[1:])
@pytest.mark.parametrize("n,k", [(2064, 2104), (8, 65544), (65544, 8)])
def test_large_tiles_grad_weight(n, k, dtype):
    """Experts of 0 to 1000 rows; weights in full and cut tiles, and of few rows or columns."""
    sizes = [1000, 1, 0, 129, 256] if n * k < 1 << 20 else [520, 0, 330]
    offsets = _offsets(sizes, 2)
    rows = max(int(offsets[-1]) + 5, 768 * len(sizes))
    g, x = _ints((rows, n), 4, dtype, n), _ints((rows, k), 4, dtype, k)
    got = K.grouped_linear_grad_weight(g.cuda(), x.cuda(), offsets.cuda()).cpu()
    want = _rounded(products.grouped_linear_grad_weight(_np(g), _np(x), offsets.numpy()), dtype)
    assert torch.equal(got, want), (got != want).nonzero()[:4].tolist()


@pytest.mark.parametrize("per", [1, 8, 9, 16, 17, 32, 33, 64, 127, 129])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_rows_a_group(per, dtype):
    """Either side of the average group sizes that other kernels take, with uneven groups."""
    sizes = [0, 2 * per, per, per + 1, per - 1]
    _check_ints(sizes, 200, 264, dtype, seed=per)
    _check_ints(sizes, 67, 75, dtype, seed=per)
    _check_ints([per], 100, 136, dtype, seed=per)
    if per in (16, 32, 33):  # with tiles enough
        _check_ints(sizes, 8200, 72, dtype, seed=per)


def test_large_tiles_twice_alike():
    """No order of the sums depends on the launch: two calls agree bit for bit."""
    x, w = _normal((2600, 1000), torch.bfloat16, 1).cuda(), _normal((1, 5208, 1000), torch.bfloat16, 2).cuda()
    o = torch.tensor([0, 2600], device="cuda")
    y = K.grouped_linear(x, w, o)
    assert torch.equal(y, K.grouped_linear(x, w, o))
    gw = K.grouped_linear_grad_weight(y, x, o)
    assert torch.equal(gw, K.grouped_linear_grad_weight(y, x, o))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sizes,n,k", [([2000], 1032, 1064), ([700, 900], 900, 1000), ([40] * 8, 2056, 136),
                                       ([130, 0, 300], 1001, 517), ([33] * 64, 40, 48)],
                         ids=lambda v: "x".join(map(str, v))[:20] if isinstance(v, list) else str(v))
def test_few_tiles_and_many(sizes, n, k, dtype):
    """Either side of where smaller tiles are taken."""
    _check_ints(sizes, n, k, dtype, seed=n)


# 16-bit tiles of 128 x 128: 192 of them and more, groups too small for the largest. On average at most 96 rows a group
# (whole rows: weights read past the caches) and more; cut rows of tiles, groups of none and of one row.
MIDDLE = {"small groups": [130, 0, 250, 1, 20], "large groups": [300, 130, 0, 77, 100]}
# Contracted lengths: one step of 128 bytes and of 64 and parts of them, odd and even numbers of steps.
WHOLE, ODD = [8, 64, 136, 200], [9, 31, 33, 133, 161]


def _check_middle(op, sizes, cols, length, dtype, off=0):
    """One operator of `cols` output columns against float64, from buffers that begin `off` elements past a vector."""
    offsets = _offsets(sizes, 2)
    rows = int(offsets[-1]) + 40
    a = _ints((rows, length), 4, dtype, cols + length)
    w = _ints((len(sizes), *((cols, length) if op == "linear" else (length, cols))), 4, dtype, cols)

    def moved(t):
        b = torch.empty(t.numel() + off, dtype=dtype, device="cuda")
        b[off:] = t.reshape(-1).cuda()
        return b[off:].view(t.shape)

    name = {"linear": "grouped_linear", "grad_input": "grouped_linear_grad_input"}[op]
    got = getattr(K, name)(moved(a), moved(w), offsets.cuda()).cpu()
    want = _rounded(getattr(products, name)(_np(a), _np(w), offsets.numpy()), dtype)
    assert torch.equal(got, want), (got != want).nonzero()[:4].tolist()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("length", WHOLE)
@pytest.mark.parametrize("groups", MIDDLE)
@pytest.mark.parametrize("op", ["linear", "grad_input"])
def test_middle_tiles(op, groups, length, dtype):
    _check_middle(op, MIDDLE[groups], 8200, length, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("length,cols", [*((n, 8203) for n in ODD), (64, 8203), (133, 8197), (133, 8200), (133, 8321)])
@pytest.mark.parametrize("groups", MIDDLE)
@pytest.mark.parametrize("op", ["linear", "grad_input"])
def test_middle_tiles_of_odd_widths(op, groups, length, cols, dtype):
    """The last column tile has 11, 5, 8 and 1 columns: less than a vector and more."""
    _check_middle(op, MIDDLE[groups], cols, length, dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("off", [1, 2, 5])
@pytest.mark.parametrize("op", ["linear", "grad_input"])
def test_middle_tiles_of_unaligned_buffers(op, off, dtype):
    _check_middle(op, MIDDLE["large groups"], 8200, 136, dtype, off=off)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("sizes,n,k", [([200, 0, 333], 1003, 1029), ([40, 0, 65, 1], 1029, 1001), ([130, 7], 1000, 1032),
                                       ([64, 63, 0, 65], 1032, 1048)], ids=lambda v: str(v)[:16])
def test_middle_tiles_grad_weight(sizes, n, k, dtype):
    """96 tiles of 128 x 128 and more: whole vectors and odd widths, steps cut at every part."""
    _check_ints(sizes, n, k, dtype, seed=k)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n,k", [(2056, 136), (2051, 133), (2056, 1032), (2051, 1029), (2057, 600)])
def test_few_rows_of_many_columns(n, k, dtype):
    """At most 8 rows a group and columns enough for every CU: whole rows and odd ones, and more steps than waves."""
    _check_ints([1, 0, 8, 3, 9], n, k, dtype, seed=k, first=1, rows=24)
