"""The expert and MXFP4 products as programs use them: on another stream than the
default one, on several at once, captured in a graph and replayed with new
inputs, and past 2^31 elements. What each computes is compared with float64 in
test_grouped_linear_gpu.py and test_mxfp4_gpu.py; here mostly with its own
ordinary call, bit for bit (no sum's order depends on the launch)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from custom_cuda_kernals_amd._lib import native

pytestmark = pytest.mark.gpu

SPIN_CYCLES = 20_000_000  # ~10 ms
OPS = ["linear", "grad_input", "grad_weight", "quant", "dequant", "mxfp4", "mxfp4_dense", "offsets"]
# Groups' sizes: a few rows each, small tiles, 128 x 128 tiles, 256 x 256 tiles (with 4200 columns).
SIZES = {"few": [2, 0, 1, 5], "small": [60, 0, 33, 70], "middle": [500, 7, 0, 1030], "wide": [2100, 0, 1300, 700]}


@pytest.fixture(autouse=True)
def _free_device_memory():
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def _randn(*shape, seed, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def _offsets(sizes):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int64, device="cuda")


def _inputs(op, sizes, seed, n=4200, k=264):
    """Device inputs of the op; every seed has the shapes of the same sizes' sum."""
    rows, experts = sum(sizes), len(sizes)
    if op == "offsets":
        g = torch.Generator().manual_seed(seed)
        return [torch.randint(0, 40, (rows, 4), generator=g).cuda()]
    x, g, w = _randn(rows, k, seed=seed), _randn(rows, n, seed=seed + 1), _randn(experts, n, k, seed=seed + 2)
    if op == "linear":
        return [x, w, _offsets(sizes)]
    if op == "grad_input":
        return [_randn(rows, k, seed=seed), _randn(experts, k, n, seed=seed + 2), _offsets(sizes)]
    if op == "grad_weight":
        return [g, x, _offsets(sizes)]
    if op == "quant":
        return [x]
    if op == "dequant":
        return [*K.mxfp4_quant(x)]
    return [*K.mxfp4_quant(x), *K.mxfp4_quant(w if op == "mxfp4" else w[0])] + (
        [_offsets(sizes)] if op == "mxfp4" else [])


def _run(op, a):
    if op == "offsets":
        return K.compute_permutation(a[0], 40, return_offsets=True)
    if op == "dequant":
        return (K.mxfp4_dequant(*a, 264, torch.bfloat16),)
    fn = {"linear": K.grouped_linear, "grad_input": K.grouped_linear_grad_input,
          "grad_weight": K.grouped_linear_grad_weight, "quant": K.mxfp4_quant, "mxfp4": K.mxfp4_linear,
          "mxfp4_dense": K.mxfp4_linear}[op]
    out = fn(*a)
    return out if isinstance(out, tuple) else (out,)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _same(got, want):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.shape == b.shape and torch.equal(_bytes(a), _bytes(b))


@pytest.mark.parametrize("op", OPS)
def test_side_stream(op):
    """The launch is on the current stream: inputs written there before the call are what it reads."""
    a = _inputs(op, SIZES["small"], 1)
    want = _run(op, a)
    late = [torch.zeros_like(t) for t in a]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(SPIN_CYCLES)
        for dst, src in zip(late, a):
            _bytes(dst).copy_(_bytes(src))
        got = _run(op, late)
        launched_on = native._last_launch_stream()
    assert launched_on == side.cuda_stream != torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    _same(got, want)


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("op", OPS)
def test_captured_and_replayed(op, size):
    """A captured call replayed with new inputs, among them other group sizes of the same sum; with the program's own
    eager calls and waits between the replays."""
    sizes = SIZES[size]
    a = _inputs(op, sizes, 3)
    _run(op, a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _run(op, a)
    for seed, order in ((11, sizes), (12, sizes[::-1]), (13, [sum(sizes)] + [0] * (len(sizes) - 1)), (11, sizes)):
        new = _inputs(op, order, seed)
        want = _run(op, new)  # eager, between the replays
        for dst, src in zip(a, new):
            _bytes(dst).copy_(_bytes(src))
        for t in out:
            _bytes(t).fill_(0xEE)
        graph.replay()
        torch.cuda.synchronize()
        _same(out, want)


@pytest.mark.parametrize("op", OPS)
def test_two_streams_at_once(op):
    a, b = _inputs(op, SIZES["middle"], 5), _inputs(op, SIZES["middle"], 6)
    want_a, want_b = _run(op, a), _run(op, b)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s, inputs in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(_run(op, inputs))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        _same(g, (want_a, want_b)[i % 2])


def test_layer_in_one_graph():
    """Router, permutation, gather, gate, up and down products and combine as one graph, replayed with other tokens
    and so other routes."""
    tokens, hidden, inner, experts, top = 300, 256, 520, 8, 2
    wg, wu, wd = (_randn(experts, *s, seed=i) for i, s in enumerate([(inner, hidden), (inner, hidden), (hidden, inner)]))

    def layer(x, logits):
        weights, ids = K.moe_router(logits, top)
        perm, unperm, offsets = K.compute_permutation(ids, experts, return_offsets=True)
        rows = K.token_gather(x, perm)
        h = K.swiglu(K.grouped_linear(rows, wg, offsets), K.grouped_linear(rows, wu, offsets))
        return K.token_combine(K.grouped_linear(h, wd, offsets), unperm, weights)

    x, logits = _randn(tokens, hidden, seed=7), _randn(tokens, experts, seed=8, dtype=torch.float32)
    layer(x, logits)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x, logits)
    for seed in (20, 21, 22):
        nx, nl = _randn(tokens, hidden, seed=seed), _randn(tokens, experts, seed=seed + 50, dtype=torch.float32)
        nl[:, seed % experts] += 4.0  # one expert liked by most
        want = layer(nx, nl)
        x.copy_(nx)
        logits.copy_(nl)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def _some(total, count, seed):
    """Rows at the start, at the end and between."""
    g = np.random.default_rng(seed)
    return sorted({0, 1, total // 2, total - 2, total - 1, *g.integers(0, total, count).tolist()})


def test_output_past_2_31_elements():
    """y and grad_x of 2.4e9 elements; rows of small integers, whose products are exact."""
    rows, n, k = 300_000, 8200, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randint(-4, 5, (rows, k), generator=g, device="cuda").bfloat16()
    w = torch.randint(-4, 5, (3, n, k), generator=g, device="cuda").bfloat16()
    o = torch.tensor([5, 5, 180_000, rows - 7], device="cuda")
    pick = _some(rows, 200, 1)
    at = torch.tensor(pick, device="cuda")
    group = torch.bucketize(at, o, right=True) - 1

    def want(weight):  # [3][cols][k] values
        y = torch.stack([x[i].double() @ weight[e].double().T if 0 <= e < 3 else
                         torch.zeros(n, dtype=torch.float64, device="cuda") for i, e in zip(pick, group.tolist())])
        return y.bfloat16()

    y = K.grouped_linear(x, w, o)
    assert y.numel() > 1 << 31 and torch.equal(y[at], want(w))
    del y
    wt = w.transpose(1, 2).contiguous()
    gx = K.grouped_linear_grad_input(x, wt, o)
    assert gx.numel() > 1 << 31 and torch.equal(gx[at], want(w))


def test_weights_past_2_31_elements():
    """40 experts of 8192 x 8192: read by the product of few rows and by a product of many, and written by the
    gradient."""
    experts, n, k = 40, 8192, 8192
    g = torch.Generator(device="cuda").manual_seed(0)
    # +-1 and 0: sums of 8192 products of at most 4 stay below 2^24
    w = torch.randint(-1, 2, (experts, n, k), generator=g, device="cuda", dtype=torch.int8).bfloat16()
    assert w.numel() > 1 << 31
    for per in (1, 40):
        x = torch.randint(-4, 5, (experts * per, k), generator=g, device="cuda").bfloat16()
        o = torch.arange(0, experts + 1, device="cuda") * per
        y, gx = K.grouped_linear(x, w, o), K.grouped_linear_grad_input(x, w, o)
        for e in (0, 31, 32, 39):
            part = x[e * per:(e + 1) * per].double()
            assert torch.equal(y[e * per:(e + 1) * per], (part @ w[e].double().T).bfloat16()), (per, e)
            assert torch.equal(gx[e * per:(e + 1) * per], (part @ w[e].double()).bfloat16()), (per, e)
    del w, y, gx
    gw = K.grouped_linear_grad_weight(x, x, o)
    assert gw.numel() > 1 << 31
    for e in (0, 31, 32, 39):
        part = x[e * per:(e + 1) * per].double()
        assert torch.equal(gw[e], (part.T @ part).bfloat16()), e


def test_more_tiles_than_a_launch_has_room_for():
    """Sizes of 2^32 threads and more (2^24 tiles of 256), which take several launches: rows, an expert's columns in
    the product of few rows, and weights. Small integers, whose sums are exact."""
    g = torch.Generator(device="cuda").manual_seed(0)
    ints = lambda *shape: torch.randint(-4, 5, shape, generator=g, device="cuda", dtype=torch.int8)
    # 2^30 + 70 rows of 4 float32: 2^24 + 2 tiles of 64 x 64
    rows = (1 << 30) + 70
    x = torch.empty(rows, 4, device="cuda")
    for part in x.split(1 << 27):
        part.copy_(ints(*part.shape))
    w = ints(3, 4, 4).float()
    cuts = [3, 1 << 29, 1 << 29, rows - 5]
    o = torch.tensor(cuts, device="cuda")
    for fn, weight in ((K.grouped_linear, w.transpose(1, 2)), (K.grouped_linear_grad_input, w)):  # [e][contracted][out]
        y = fn(x, w, o)
        assert (y[:3] == 0).all() and (y[rows - 5:] == 0).all()
        for e in (0, 2):
            for first in range(cuts[e], cuts[e + 1], 1 << 27):
                part = slice(first, min(first + (1 << 27), cuts[e + 1]))
                want = sum(x[part, c, None] * weight[e, c] for c in range(4))
                assert torch.equal(y[part], want), (e, first)
        del y, want
    del x
    torch.cuda.empty_cache()
    # 1024 experts of 4 x 2^20 weights: 2^24 tiles
    experts, wide = 1024, 1 << 20
    x, gy = ints(20, wide).float(), ints(20, 4).float()
    o = torch.zeros(experts + 1, dtype=torch.int64)
    o[1:], o[600:], o[1024:] = 7, 13, 20  # experts 0, 599 and 1023 have rows
    o = o.cuda()
    gw = K.grouped_linear_grad_weight(gy, x, o)
    for e, part in ((0, slice(0, 7)), (599, slice(7, 13)), (1023, slice(13, 20))):
        assert torch.equal(gw[e], sum(gy[s, :, None] * x[s] for s in range(part.start, part.stop))), e
        gw[e] = 0
    assert not any(bool(part.any()) for part in gw.split(128))
    del x, gw
    torch.cuda.empty_cache()
    # 700 experts of 2^21 x 8 half weights: 700 x 65536 tiles of 16 x 32
    experts, n = 700, 1 << 21
    w = ints(experts, n, 8).half()
    x = ints(experts, 8).half()
    y = K.grouped_linear(x, w, torch.arange(experts + 1, device="cuda"))
    for e in (0, 1, 255, 256, 511, 512, 698, 699):
        assert torch.equal(y[e], (x[e].float() * w[e].float()).sum(-1).half()), e


def test_mxfp4_past_2_31_elements():
    rows, k = 540_000, 4096
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda")
    for part in x.split(60_000):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    codes, scales = K.mxfp4_quant(x)
    assert x.numel() > 1 << 31
    at = torch.tensor(_some(rows, 300, 2), device="cuda")
    few = K.mxfp4_quant(x[at])
    _same((codes[at], scales.view(torch.uint8)[at]), (few[0], few[1].view(torch.uint8)))
    back = K.mxfp4_dequant(codes, scales, k, torch.bfloat16)
    assert torch.equal(back[at], K.mxfp4_dequant(*few, k, torch.bfloat16))
    del x, back
    w = K.mxfp4_quant(_randn(4200, k, seed=3))
    y = K.mxfp4_linear(codes, scales, *w)
    assert y.numel() > 1 << 31
    # Another kernel does the few: alike up to the rounding of the sums (4096 products: (k + 2) 2^-24 of the
    # magnitudes' sum each) and a step of the result.
    one = K.mxfp4_linear(*few, *w).double()
    xv, wv = K.mxfp4_dequant(*few, k, torch.float32).abs().double(), K.mxfp4_dequant(*w, k, torch.float32).abs().double()
    bound = 2 * (k + 2) * 2.0 ** -24 * (xv @ wv.T) + 2.0 ** -7 * one.abs()
    assert ((y[at].double() - one).abs() <= bound).all()


@pytest.mark.parametrize("op", ["grouped_linear", "mxfp4"])
def test_cli_targets(op):
    """What `compare` and `profile` call: kernel and formula agree up to the formula's own roundings (bf16 products'
    sums and results, so a step of 2^-7 of the largest magnitude covers both)."""
    from custom_cuda_kernals_amd.cli.registry import REGISTRY

    target = REGISTRY[op].build_target("cuda")
    got, want = target.kernel().double(), target.eager().double()
    assert got.shape == want.shape
    assert (got - want).abs().max() <= 2.0 ** -7 * want.abs().max()


@pytest.mark.parametrize("groups", [1024, 1000])
def test_offsets_in_no_order_of_many_groups(groups):
    """As many groups as are taken, each of them as long as the rows or of none in turn: every tile named is inside,
    and the calls end; nothing behind the outputs is written."""
    rows, n, k = 5000, 64, 64
    o = torch.zeros(groups + 1, dtype=torch.int64)
    o[1::2] = rows
    o = o.cuda()
    buffers = [torch.full((size + 4096,), 55, dtype=torch.bfloat16, device="cuda")
               for size in (rows * n, rows * k, groups * n * k)]
    x, g, w = _randn(rows, k, seed=1), _randn(rows, n, seed=2), _randn(groups, n, k, seed=3)
    native.grouped_linear_fwd(x, w, o, buffers[0][:rows * n].view(rows, n))
    native.grouped_linear_grad_input(g, w, o, buffers[1][:rows * k].view(rows, k))
    native.grouped_linear_grad_weight(g, x, o, buffers[2][:groups * n * k].view(groups, n, k))
    torch.cuda.synchronize()
    for b in buffers:
        assert (b[-4096:] == 55).all()
