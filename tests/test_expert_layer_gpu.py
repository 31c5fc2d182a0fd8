"""The MoE dispatch and the expert products as a layer uses them: router,
permutation with the experts' offsets, gather, gate and up products, SwiGLU, down
product, combine; with the products' gradients; and the same in MXFP4. Each
product is compared with float64 on the inputs it was given (bounds as in
test_grouped_linear_gpu.py); the other steps are compared bit for bit elsewhere."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from oracle import moe, products

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _randn(*shape, seed, dtype=torch.bfloat16, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


def _np(t):
    return t.double().cpu().numpy()


def _close(got, exact, magnitude, length, what):
    sum_error = (length + 2) * U * magnitude
    bound = sum_error + torch.finfo(got.dtype).eps / 2 * (np.abs(exact) + sum_error) + torch.finfo(got.dtype).tiny
    assert (np.abs(_np(got) - exact) <= bound).all(), what


def _check(got, fn, a, b, offsets, length, what):
    a, b, o = _np(a), _np(b), offsets.cpu().numpy()
    _close(got, fn(a, b, o), fn(np.abs(a), np.abs(b), o), length, what)


@pytest.mark.parametrize("ids,experts", [("spread", 8), ("one", 8), ("outside", 6), ("spread", 256)])
@pytest.mark.parametrize("tokens,k", [(1, 1), (37, 2), (700, 6), (16384, 4)])
def test_offsets(tokens, k, experts, ids):
    """Every expert's run of sorted entries, with ids outside the experts behind them all; in one launch and in
    three, the two index tensors as without the offsets."""
    g = torch.Generator().manual_seed(tokens)
    t = torch.randint(0, experts, (tokens, k), generator=g)
    if ids == "one":
        t.fill_(experts - 2)
    if ids == "outside":
        t = torch.randint(-2, experts + 3, (tokens, k), generator=g)
    perm, unperm, offsets = K.compute_permutation(t.cuda(), experts, return_offsets=True)
    two = K.compute_permutation(t.cuda(), experts)
    assert torch.equal(perm, two[0]) and torch.equal(unperm, two[1])
    inside = t[(t >= 0) & (t < experts)]
    want = np.concatenate([[0], np.cumsum(np.bincount(inside.numpy(), minlength=experts))])
    assert offsets.dtype == torch.int64 and np.array_equal(offsets.cpu().numpy(), want)


def test_offsets_without_entries():
    perm, unperm, offsets = K.compute_permutation(torch.zeros(0, 2, dtype=torch.int64, device="cuda"), 5,
                                                  return_offsets=True)
    assert perm.shape == (0,) and unperm.shape == (0, 2) and torch.equal(offsets.cpu(), torch.zeros(6, dtype=torch.int64))


@pytest.mark.parametrize("tokens,experts,top_k,hidden,ffn", [(1, 8, 2, 64, 96), (90, 8, 2, 256, 520), (61, 40, 6, 136, 72),
                                                             (300, 3, 3, 100, 75)])
def test_layer_and_its_gradients(tokens, experts, top_k, hidden, ffn):
    x = _randn(tokens, hidden, seed=0)
    w_gate, w_up = (_randn(experts, ffn, hidden, seed=s, std=hidden ** -0.5) for s in (1, 2))
    w_down = _randn(experts, hidden, ffn, seed=3, std=ffn ** -0.5)
    weights, ids = K.moe_router(_randn(tokens, experts, seed=4, dtype=torch.float32), top_k)
    perm, unperm, offsets = K.compute_permutation(ids, experts, return_offsets=True)
    rows = K.token_gather(x, perm)
    gate, up = K.grouped_linear(rows, w_gate, offsets), K.grouped_linear(rows, w_up, offsets)
    act = K.swiglu(gate, up)
    down = K.grouped_linear(act, w_down, offsets)
    out = K.token_combine(down, unperm, weights)
    _check(gate, products.grouped_linear, rows, w_gate, offsets, hidden, "gate")
    _check(up, products.grouped_linear, rows, w_up, offsets, hidden, "up")
    _check(down, products.grouped_linear, act, w_down, offsets, ffn, "down")
    assert torch.equal(out.cpu(), moe.token_combine(down.cpu(), unperm.cpu(), weights.cpu()))
    grad = _randn(*down.shape, seed=5)
    g_act = K.grouped_linear_grad_input(grad, w_down, offsets)
    g_down = K.grouped_linear_grad_weight(grad, act, offsets)
    _check(g_act, products.grouped_linear_grad_input, grad, w_down, offsets, hidden, "grad_act")
    _check(g_down, products.grouped_linear_grad_weight, grad, act, offsets, int(offsets.diff().max()), "grad_down")


@pytest.mark.parametrize("tokens,experts,top_k,hidden,ffn", [(3, 8, 2, 64, 96), (150, 8, 2, 256, 320), (64, 40, 5, 160, 72)])
def test_layer_in_mxfp4(tokens, experts, top_k, hidden, ffn):
    """Tokens quantised once, before the gather moves their codes and scales; the
    activation quantised by row."""
    x = _randn(tokens, hidden, seed=0)
    w_up = _randn(experts, ffn, hidden, seed=1, std=hidden ** -0.5)
    w_down = _randn(experts, hidden, ffn, seed=3, std=ffn ** -0.5)
    weights, ids = K.moe_router(_randn(tokens, experts, seed=4, dtype=torch.float32), top_k)
    perm, unperm, offsets = K.compute_permutation(ids, experts, return_offsets=True)
    codes, scales = K.mxfp4_quant(x)
    rows_c = K.token_gather(codes.view(torch.float8_e4m3fn), perm).view(torch.uint8)
    rows_s = K.token_gather(scales.view(torch.float8_e4m3fn), perm).view(torch.float8_e8m0fnu)
    up_w, down_w = K.mxfp4_quant(w_up), K.mxfp4_quant(w_down)
    up = K.mxfp4_linear(rows_c, rows_s, *up_w, offsets)
    act = K.mxfp4_quant(K.swiglu(up, up))
    down = K.mxfp4_linear(*act, *down_w, offsets)
    values = lambda pair, k: K.mxfp4_dequant(*pair, k, torch.float32)
    assert torch.equal(values((rows_c, rows_s), hidden), values((codes, scales), hidden)[perm])
    _check(up, products.grouped_linear, values((rows_c, rows_s), hidden), values(up_w, hidden), offsets, hidden, "up")
    _check(down, products.grouped_linear, values(act, ffn), values(down_w, ffn), offsets, ffn, "down")
    out = K.token_combine(down, unperm, weights)
    assert torch.equal(out.cpu(), moe.token_combine(down.cpu(), unperm.cpu(), weights.cpu()))
