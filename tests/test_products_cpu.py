"""The expert products and MXFP4 on the CPU: what the launchers and the binding
refuse, empty work, the one-call functions' argument handling, and the float64
restatement of MXFP4 (oracle/products.py) against the format's table."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from custom_cuda_kernals_amd._lib import native
from oracle import products
from tests import _cck
from tests.test_abi_cpu import F

I64, U8, E8, F32 = torch.int64, torch.uint8, torch.float8_e8m0fnu, torch.float32


def test_empty_work_returns_success_without_device_calls():
    lib = _cck.load()
    assert lib.launch_grouped_linear_fwd(None, None, None, None, 0, 8, 16, 16, 2, None) == 0
    assert lib.launch_grouped_linear_fwd(None, None, None, None, 4, 8, 0, 16, 2, None) == 0
    assert lib.launch_grouped_linear_grad_input(None, None, None, None, 4, 8, 16, 0, 2, None) == 0
    assert lib.launch_grouped_linear_grad_weight(None, None, None, None, 4, 8, 0, 16, 2, None) == 0
    assert lib.launch_mxfp4_quant_fwd(None, None, None, 0, 16, 2, None) == 0
    assert lib.launch_mxfp4_dequant_fwd(None, None, None, 4, 0, 2, None) == 0
    assert lib.launch_mxfp4_linear_fwd(None, None, None, None, None, None, 0, 1, 16, 4, 2, None) == 0
    assert lib.launch_mxfp4_linear_fwd(None, None, None, None, None, None, 4, 1, 16, 0, 2, None) == 0


@pytest.mark.parametrize("name", ["fwd", "grad_input", "grad_weight"])
def test_product_launchers_refuse_before_device_calls(name):
    fn = getattr(_cck.load(), f"launch_grouped_linear_{name}")
    for rows, experts, n, k, dtype in [(4, 8, 16, 16, 3), (4, 8, 16, 16, 9),  # not a compute dtype
                                       (4, 1025, 16, 16, 2), (1 << 31, 8, 16, 16, 2),
                                       (4, 8, (1 << 21) + 1, 16, 2), (4, 8, 16, (1 << 21) + 1, 2),
                                       (4, 8, 16, (1 << 20) + 1, 0)]:
        assert fn(None, None, None, None, rows, experts, n, k, dtype, None) == 1
    if name == "grad_weight":
        assert fn(None, None, None, None, -1, 8, 16, 16, 2, None) == 1
    else:
        assert fn(None, None, None, None, 4, 0, 16, 16, 2, None) == 1


def test_mxfp4_launchers_refuse_before_device_calls():
    lib = _cck.load()
    assert lib.launch_mxfp4_quant_fwd(None, None, None, 4, 16, 3, None) == 1
    assert lib.launch_mxfp4_quant_fwd(None, 2, None, 4, 16, 2, None) == 1  # codes not 4-byte aligned
    assert lib.launch_mxfp4_quant_fwd(None, None, None, 4, 1 << 31, 2, None) == 1
    assert lib.launch_mxfp4_quant_fwd(None, None, None, 1 << 40, 1 << 30, 2, None) == 1
    assert lib.launch_mxfp4_dequant_fwd(None, None, None, 4, 16, 4, None) == 1
    assert lib.launch_mxfp4_dequant_fwd(None, None, None, 4, 1 << 31, 2, None) == 1
    lin = lib.launch_mxfp4_linear_fwd
    assert lin(None, None, None, None, None, None, 4, 1, 16, 4, 7, None) == 1
    assert lin(None, None, None, None, None, None, 4, 2, 16, 4, 2, None) == 1  # experts without offsets
    assert lin(None, None, None, None, None, None, 1 << 31, 1, 16, 4, 2, None) == 1
    assert lin(None, None, None, None, None, None, 4, 1, 16, (1 << 18) + 1, 2, None) == 1
    assert lin(None, None, None, None, 8, None, 4, 1025, 16, 4, 2, None) == 1


NO_DEVICE = 100  # hipErrorNoDevice: the launcher took the sizes and went on to the launch


@pytest.mark.skipif(torch.cuda.is_available(), reason="without operands the launch must not happen")
@pytest.mark.parametrize("name,rows,experts,n,k,dtype", [
    ("fwd", 1 << 30, 2, 4, 4, 0), ("fwd", (1 << 31) - 1, 2, 4, 4, 0), ("fwd", (1 << 31) - 1, 2, 8, 8, 2),
    ("fwd", 8192, 1024, 1 << 21, 8, 1), ("grad_input", 1 << 30, 2, 4, 4, 0), ("grad_input", (1 << 31) - 1, 2, 8, 8, 1),
    ("grad_weight", 1, 1024, 4, 1 << 20, 0), ("grad_weight", 1, 1024, 1 << 20, 4, 0),
    ("grad_weight", 1 << 20, 1024, 8192, 8192, 2)])
def test_more_tiles_than_a_launch_has_room_for(name, rows, experts, n, k, dtype):
    """Sizes of 2^32 threads and more, whose operands a card holds."""
    fn = getattr(_cck.load(), f"launch_grouped_linear_{name}")
    assert fn(None, None, None, None, rows, experts, n, k, dtype, None) == NO_DEVICE


@pytest.mark.skipif(torch.cuda.is_available(), reason="without operands the launch must not happen")
@pytest.mark.parametrize("rows,experts,n,blocks", [((1 << 31) - 1, 1, 16, 4), ((1 << 31) - 1, 1, 8, 1),
                                                   (8192, 1024, 1 << 21, 1)])
def test_more_mxfp4_tiles_than_a_launch_has_room_for(rows, experts, n, blocks):
    lin = _cck.load().launch_mxfp4_linear_fwd
    offsets = 8 if experts > 1 else None
    assert lin(None, None, None, None, offsets, None, rows, experts, n, blocks, 2, None) == NO_DEVICE


@pytest.mark.skipif(torch.cuda.is_available(), reason="the output is no memory of a device")
def test_sums_of_nothing_are_written():
    """A product over no elements has an output all the same: the launcher goes on to the launch."""
    lib = _cck.load()
    assert lib.launch_grouped_linear_fwd(None, None, 8, 64, 4, 8, 16, 0, 2, None) == NO_DEVICE
    assert lib.launch_grouped_linear_grad_input(None, None, 8, 64, 4, 8, 0, 16, 2, None) == NO_DEVICE
    assert lib.launch_mxfp4_linear_fwd(None, None, None, None, None, 64, 4, 1, 16, 0, 2, None) == NO_DEVICE


def test_more_tiles_than_any_card_holds():
    lib = _cck.load()
    assert lib.launch_grouped_linear_fwd(None, None, None, None, (1 << 31) - 1, 2, 1 << 20, 8, 0, None) == 1
    assert lib.launch_grouped_linear_grad_input(None, None, None, None, (1 << 31) - 1, 2, 8, 1 << 20, 0, None) == 1
    assert lib.launch_grouped_linear_grad_weight(None, None, None, None, 1, 1024, 1 << 20, 1 << 20, 0, None) == 1


def _raises(fn, *args, match):
    with pytest.raises(ValueError, match=match):
        fn(*args)


def test_grouped_linear_checks():
    f = native.grouped_linear_fwd
    x, w, o, y = F(6, 8), F(2, 4, 8), F(3, dtype=I64), F(6, 4)
    _raises(f, F(6, 8, device="cpu"), w, o, y, match="'x' must be a CUDA tensor")
    _raises(f, x, F(2, 4, 8, contiguous=False), o, y, match="'weight' must be contiguous")
    _raises(f, x, w, F(3, dtype=torch.int32), y, match="offsets must be int64")
    _raises(f, F(6, 8, dtype=torch.float8_e4m3fn), w, o, y, match="x is F8E4M3")
    _raises(f, x, F(2, 4, 8, dtype=F32), o, y, match="'weight' is F32 but expected BF16")
    _raises(f, x, w, o, F(6, 4, dtype=F32), match="'y' is F32")
    _raises(f, F(6, 2, 4), w, o, y, match="x must be 2-D")
    _raises(f, x, w, F(1, dtype=I64), y, match="offsets must be 1-D")
    _raises(f, x, w, F(1026, dtype=I64), y, match="offsets must be 1-D")
    _raises(f, x, w, F(4, dtype=I64), y, match=r"weight must be \[num_experts, n, k\] = \[3, n, 8\]")
    _raises(f, x, F(2, 4, 9), o, y, match="weight must be")
    _raises(f, x, F(4, 8), o, y, match="weight must be")
    _raises(f, x, w, o, F(6, 5), match=r"y shape \[6, 5\] must be \[6, 4\]")
    k = (1 << 21) + 8
    _raises(f, F(6, k), F(2, 4, k), o, y, match="more than 4 MiB")
    _raises(f, F(1 << 31, 8), w, o, F(1 << 31, 4), match=r"more than 2\^31 - 1 rows")
    g = native.grouped_linear_grad_input
    _raises(g, F(6, 5), w, o, F(6, 8), match=r"= \[2, 5, k\]")
    _raises(g, F(6, 4), w, o, F(6, 9), match="grad_x shape")
    _raises(g, F(6, 4), w, o, F(6, 8, dtype=torch.float16), match="'grad_x' is F16")
    h = native.grouped_linear_grad_weight
    _raises(h, F(6, 4), F(7, 8), o, F(2, 4, 8), match="same rows")
    _raises(h, F(6, 4), F(6, 8), o, F(3, 4, 8), match=r"grad_weight shape \[3, 4, 8\] must be \[2, 4, 8\]")
    _raises(h, F(6, 4), F(6, 8, dtype=F32), o, F(2, 4, 8), match="'x' is F32")


def test_devices_must_agree():
    other = F(3, dtype=I64)
    other.device.index = 1
    _raises(native.grouped_linear_fwd, F(6, 8), F(2, 4, 8), other, F(6, 4), match="device mismatch: 'offsets' is on cuda:1")
    codes = F(4, 16, dtype=U8)
    codes.device.index = 2
    _raises(native.mxfp4_quant_fwd, F(4, 32), codes, F(4, 1, dtype=E8), match="'codes' is on cuda:2")


def test_mxfp4_checks():
    q = native.mxfp4_quant_fwd
    _raises(q, F(4, 40, dtype=I64), F(4, 32, dtype=U8), F(4, 2, dtype=E8), match="unsupported dtype")
    _raises(q, F(4, 40), F(4, 32), F(4, 2, dtype=E8), match="codes must be uint8")
    _raises(q, F(4, 40), F(4, 32, dtype=U8), F(4, 2, dtype=U8), match="scales must be float8_e8m0fnu")
    _raises(q, F(4, 40), F(4, 16, dtype=U8), F(4, 1, dtype=E8), match=r"codes shape \[4, 16\] must be \[4, 32\]")
    _raises(q, F(4, 40), F(4, 32, dtype=U8), F(4, 3, dtype=E8), match="do not belong together")
    _raises(q, F(), F(dtype=U8), F(dtype=E8), match="at least 1 dimension")
    d = native.mxfp4_dequant_fwd
    _raises(d, F(4, 32, dtype=U8), F(4, 2, dtype=E8), F(4, 65), match="codes shape")
    _raises(d, F(4, 32, dtype=U8), F(4, 2, dtype=E8), F(4, 40, dtype=torch.float8_e5m2), match="out is F8E5M2")
    f = native.mxfp4_linear_fwd
    c, s, y = F(4, 32, dtype=U8), F(4, 2, dtype=E8), F(4, 4)
    _raises(f, c, s, F(4, 48, dtype=U8), F(4, 3, dtype=E8), None, y, match="x_codes' blocks")
    _raises(f, c, s, F(2, 4, 32, dtype=U8), F(2, 4, 2, dtype=E8), None, y, match="without offsets")
    _raises(f, c, s, c, s, F(3, dtype=I64), y, match="num_experts, n, 16")
    _raises(f, c, s, F(3, 4, 32, dtype=U8), F(3, 4, 2, dtype=E8), F(3, dtype=I64), y, match="num_experts, n, 16")
    _raises(f, c, F(4, 3, dtype=E8), c, s, None, y, match="x codes .* do not belong together")
    _raises(f, c, s, c, s, None, F(4, 5), match="y shape")
    _raises(f, c, s, c, s, None, F(4, 4, dtype=torch.float8_e5m2), match="y is F8E5M2")


def test_permutation_offsets_checks():
    f = native.moe_permutation_offsets_fwd
    t, p = F(4, 2, dtype=I64), F(8, dtype=I64)
    _raises(f, t, p, t, F(8, dtype=I64), 8, match=r"expert_offsets shape \[8\] must be \[9\]")
    _raises(f, t, p, t, F(9, dtype=torch.int32), 8, match="expert_offsets must be int64")
    _raises(f, t, p, t, F(258, dtype=I64), 257, match=r"must be in \[1, 256\]")
    with pytest.raises(ValueError, match="return_offsets needs num_experts"):
        K.compute_permutation(torch.zeros(4, 2, dtype=I64), return_offsets=True)
    lib = _cck.load()
    assert lib.launch_moe_permutation_offsets_fwd(None, None, None, None, 4, 2, 257, None) == 1
    assert lib.launch_moe_permutation_offsets_fwd(None, None, None, None, 1 << 30, 8, 16, None) == 1


X, IDS, OFF = torch.zeros(4, 16), torch.zeros(4, 2, dtype=I64), torch.tensor([0, 4])
CODES, SCALES = torch.zeros(4, 16, dtype=U8), torch.zeros(4, 1, dtype=U8).view(E8)
CALLS = {
    "compute_permutation_offsets_call": (IDS, 8),
    "grouped_linear_call": (X, X[None], OFF),
    "grouped_linear_grad_input_call": (X, torch.zeros(1, 16, 16), OFF),
    "grouped_linear_grad_weight_call": (X, X, OFF),
    "mxfp4_quant_call": (X,),
    "mxfp4_dequant_call": (CODES, SCALES, 32, F32),
    "mxfp4_linear_call": (CODES, SCALES, CODES, SCALES, None, F32),
}


@pytest.mark.parametrize("name", CALLS)
def test_other_arguments_return_none(name):
    call, args = getattr(native, name), CALLS[name]
    assert call(*args) is None  # CPU tensors
    assert call() is None and call(*args, None) is None
    for i in range(len(args)):
        for other in (None, object(), 3, 2.5, "e4m3", 1 << 80, [1], X.numpy(), torch.int8, torch.zeros(0)):
            assert call(*args[:i], other, *args[i + 1:]) is None


def test_cpu_tensors_are_refused():
    calls = [lambda: K.grouped_linear(X, X[None], OFF), lambda: K.grouped_linear_grad_input(X, X[None], OFF),
             lambda: K.grouped_linear_grad_weight(X, X, OFF), lambda: K.mxfp4_quant(X),
             lambda: K.mxfp4_dequant(CODES, SCALES, 32), lambda: K.mxfp4_linear(CODES, SCALES, CODES, SCALES),
             lambda: K.compute_permutation(IDS, 8, return_offsets=True)]
    for call in calls:
        with pytest.raises(ValueError, match="must be a CUDA tensor, got device type 'cpu'"):
            call()
    for call in (lambda: K.grouped_linear(X, X, OFF), lambda: K.grouped_linear_grad_weight(X, X[0], OFF),
                 lambda: K.mxfp4_linear(CODES, SCALES, CODES, SCALES, OFF), lambda: K.mxfp4_quant(X[0, 0]),
                 lambda: K.mxfp4_dequant(CODES, SCALES, -1)):
        with pytest.raises(ValueError, match="shape mismatch"):
            call()


def test_oracle_quant_against_the_table():
    """Every multiple of 1/64 in [0, 8) under a scale of 1, against the nearest table entry picked by exhaustion."""
    v = np.arange(0, 512) / 64.0
    x = np.concatenate([np.full((512, 1), 4.0), v[:, None]], axis=1)
    codes, scales = products.mxfp4_quant(x)
    assert (scales == np.where(v >= 8, 128, 127)[:, None]).all()
    for value, byte in zip(v, codes[:, 0]):
        best = min(range(8), key=lambda c: (abs(products.MAGNITUDES[c] - value), c % 2))
        assert byte >> 4 == best, value
    back = products.mxfp4_values(codes, scales, 2)
    # half a step: 1/2 below 2, 1 below 4, 2 below 6; beyond 6 what saturates
    half = np.where(v < 2, 0.25, np.where(v < 4, 0.5, np.where(v < 6, 1.0, v - 6)))
    assert (np.abs(back[:, 1] - v) <= half).all()
    assert np.isnan(products.mxfp4_values(*products.mxfp4_quant(np.array([[np.inf, 1.0]])), 2)).all()


def test_oracle_products_against_a_loop():
    rng = np.random.default_rng(0)
    x, w, g = rng.normal(size=(6, 3)), rng.normal(size=(2, 4, 3)), rng.normal(size=(6, 4))
    offsets = np.array([1, 3, 5])
    of = [None, 0, 0, 1, 1, None]
    y = np.array([[0.0 if of[s] is None else sum(x[s, k] * w[of[s], n, k] for k in range(3)) for n in range(4)]
                  for s in range(6)])
    gx = np.array([[0.0 if of[s] is None else sum(g[s, n] * w[of[s], n, k] for n in range(4)) for k in range(3)]
                   for s in range(6)])
    gw = np.array([[[sum(g[s, n] * x[s, k] for s in range(6) if of[s] == e) for k in range(3)] for n in range(4)]
                   for e in range(2)])
    assert np.allclose(products.grouped_linear(x, w, offsets), y, rtol=1e-14, atol=1e-14)
    assert np.allclose(products.grouped_linear_grad_input(g, w, offsets), gx, rtol=1e-14, atol=1e-14)
    assert np.allclose(products.grouped_linear_grad_weight(g, x, offsets), gw, rtol=1e-14, atol=1e-14)


def test_cli_names_the_products():
    from typer.testing import CliRunner

    from custom_cuda_kernals_amd.cli import app as cli_app

    run = CliRunner().invoke
    for op, entry in (("grouped_linear", "launch_grouped_linear_grad_weight"), ("mxfp4", "launch_mxfp4_linear_fwd")):
        shown = run(cli_app.app, ["info", op])
        assert shown.exit_code == 0 and entry in shown.output
        assert run(cli_app.app, ["benchmark", op, "--rerun"]).exit_code == 1  # bench.py does not time them
