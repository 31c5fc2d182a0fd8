"""Refusals of the decode step's operators, on the CPU: every call here fails its checks
before a launch. Tensors on a GPU are stood in for by attribute-only objects. Also the
frequencies of rope_frequencies, and the oracle against plain torch."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from custom_cuda_kernals_amd._lib import native
from oracle import decode
from oracle import fp8 as ofp8

BF16, F32, F64, I64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.int64, torch.float8_e4m3fn


class Device:
    def __init__(self, kind="cuda", index=0):
        self.type, self.index = kind, index


class T:
    """A tensor's attributes, contiguous unless it has strides."""

    def __init__(self, *shape, dtype=BF16, device="cuda", index=0, strides=None, ptr=1 << 20):
        self.shape, self.dtype, self.device, self._strides, self._ptr = shape, dtype, Device(device, index), strides, ptr

    def is_contiguous(self):
        return self._strides is None

    def stride(self):
        return self._strides

    def data_ptr(self):
        return self._ptr


def raises(match, fn, *args):
    with pytest.raises(ValueError, match=match):
        fn(*args)


def rope_args(**kw):
    a = {"q": T(5, 4, 64), "k": T(5, 2, 64), "positions": T(5, dtype=I64), "frequencies": T(32, dtype=F64),
         "q_out": T(5, 4, 64, ptr=2 << 20), "k_out": T(5, 2, 64, ptr=3 << 20), "layout": "half", "scale": 1.0,
         "inverse": False}
    return [{**a, **kw}[n] for n in a]


@pytest.mark.parametrize("match,kw", [
    ("layout must be", {"layout": "split"}),
    ("must be a CUDA tensor, got device type 'cpu'", {"q": T(5, 4, 64, device="cpu")}),
    ("must be a CUDA tensor, got device type 'cpu'", {"k": T(5, 2, 64, device="cpu", strides=(500, 64, 1))}),
    ("unsupported dtype 'torch.float64'", {"q": T(5, 4, 64, dtype=F64)}),
    ("unsupported dtype", {"q": T(5, 4, 64, dtype=E4M3)}),
    (r"q must be \[..., heads, head_dim\]", {"q": T(4, 64)}),
    ("'q' must be contiguous, or", {"q": T(5, 4, 64, strides=(256, 64, 2))}),
    ("'q' must be contiguous, or", {"q": T(1, 5, 4, 64, strides=(9999, 256, 64, 1))}),
    ("dtype mismatch: 'k'", {"k": T(5, 2, 64, dtype=F32)}),
    ("k must have q's tokens and head_dim", {"k": T(6, 2, 64)}),
    ("k must have q's tokens and head_dim", {"k": T(5, 2, 32)}),
    ("device mismatch: 'k'", {"k": T(5, 2, 64, index=1)}),
    ("positions must be int64", {"positions": T(5, dtype=torch.int32)}),
    ("positions shape", {"positions": T(4, dtype=I64)}),
    ("device mismatch: 'positions'", {"positions": T(5, dtype=I64, index=1)}),
    ("frequencies must be float64", {"frequencies": T(32, dtype=F32)}),
    ("at most head_dim / 2", {"frequencies": T(33, dtype=F64)}),
    ("'frequencies' is not on q's device", {"frequencies": T(32, dtype=F64, index=1)}),
    ("q_out must match q's shape", {"q_out": T(5, 5, 64)}),
    ("dtype mismatch: 'k_out'", {"k_out": T(5, 2, 64, dtype=F32)}),
    ("elements that share memory", {"q_out": T(5, 4, 64, strides=(0, 64, 1))}),
    ("elements that share memory", {"q_out": T(5, 4, 64, strides=(256, 32, 1))}),
    ("with other strides", {"q_out": T(5, 4, 64, strides=(512, 64, 1))}),
    ("are the same memory", {"q_out": T(5, 4, 64, ptr=3 << 20)}),
    ("must be at most 2048", {"q": T(5, 4, 4096), "k": T(5, 2, 4096)}),
    ("more than 2\\^20 elements", {"q": T(5, 1 << 15, 64)}),
])
def test_rope_at_refuses(match, kw):
    raises(match, native.rope_at_fwd, *rope_args(**kw))


def cache_args(**kw):
    a = {"q": T(5, 4, 64), "k": T(5, 2, 64), "v": T(5, 2, 64), "key_cache": T(3, 16, 2, 64),
         "value_cache": T(3, 16, 2, 64), "slots": T(5, dtype=I64), "positions": T(5, dtype=I64),
         "frequencies": T(32, dtype=F64), "q_out": T(5, 4, 64, ptr=2 << 20), "layout": "half", "scale": 1.0,
         "key_scale": 1.0, "value_scale": 1.0}
    return [{**a, **kw}[n] for n in a]


FP8_CACHES = {"key_cache": T(3, 16, 2, 64, dtype=E4M3), "value_cache": T(3, 16, 2, 64, dtype=E4M3)}


@pytest.mark.parametrize("match,kw", [
    ("v must have q's tokens", {"v": T(4, 2, 64)}),
    ("k and v must share", {"v": T(5, 3, 64)}),
    ("'key_cache' is F32 but expected BF16", {"key_cache": T(3, 16, 2, 64, dtype=F32)}),
    (r"key_cache must be \[pages, page_size, 2, 64\]", {"key_cache": T(3, 16, 4, 64)}),
    (r"key_cache must be \[pages, page_size, 2, 64\]", {"key_cache": T(48, 2, 64)}),
    ("page_size of 1 or more", {"key_cache": T(3, 0, 2, 64)}),
    ("must be contiguous", {"key_cache": T(3, 16, 2, 64, strides=(9999, 128, 64, 1))}),
    ("dtype mismatch: 'value_cache'", {"key_cache": T(3, 16, 2, 64, dtype=E4M3)}),
    ("must share the same shape", {"value_cache": T(4, 16, 2, 64)}),
    ("device mismatch: 'value_cache'", {"value_cache": T(3, 16, 2, 64, index=1)}),
    ("belong to an FP8 cache", {"key_scale": 0.5}),
    (r"in \[1e-30, 1e30\]", {**FP8_CACHES, "value_scale": 0.0}),
    (r"in \[1e-30, 1e30\]", {**FP8_CACHES, "key_scale": float("nan")}),
    (r"in \[1e-30, 1e30\]", {**FP8_CACHES, "key_scale": -1.0}),
    ("slots must be int64", {"slots": T(5, dtype=torch.int32)}),
    ("slots shape", {"slots": T(6, dtype=I64)}),
    ("positions shape", {"positions": T(5, 1, dtype=I64)}),
    ("device mismatch: 'slots'", {"slots": T(5, dtype=I64, index=1)}),
    ("q_out must match", {"q_out": T(5, 4, 32)}),
])
def test_rope_to_cache_refuses(match, kw):
    raises(match, native.rope_to_cache_fwd, *cache_args(**kw))


def attention_args(**kw):
    a = {"q": T(3, 8, 64), "key_cache": T(9, 16, 2, 64), "value_cache": T(9, 16, 2, 64),
         "page_table": T(3, 4, dtype=I64), "lengths": T(3, dtype=I64), "out": T(3, 8, 64), "lse": T(3, 8, dtype=F32),
         "workspace": T(1 << 20, dtype=F32), "scale": 0.1, "window": 0, "key_scale": 1.0, "value_scale": 1.0}
    return [{**a, **kw}[n] for n in a]


def _of(dim, heads=8):
    caches = T(9, 16, 2, dim)
    return {"q": T(3, heads, dim), "key_cache": caches, "value_cache": caches, "out": T(3, heads, dim)}


@pytest.mark.parametrize("match,kw", [
    (r"q must be 3-D", {"q": T(3, 1, 8, 64)}),
    (r"key_cache must be \[pages", {"key_cache": T(9, 16, 128)}),
    ("'key_cache' is F32 but expected BF16", {"key_cache": T(9, 16, 2, 64, dtype=F32)}),
    ("must be a multiple of the caches'", _of(64, heads=7)),
    ("multiple of 16", _of(72)),
    ("multiple of 16", _of(272)),
    ("page_table must be int64", {"page_table": T(3, 4, dtype=torch.int32)}),
    ("page_table must be", {"page_table": T(2, 4, dtype=I64)}),
    ("page_table must be", {"page_table": T(12, dtype=I64)}),
    ("more than 2\\^30 positions", {"page_table": T(3, 1 << 27, dtype=I64)}),
    ("lengths shape", {"lengths": T(3, 1, dtype=I64)}),
    ("device mismatch: 'lengths'", {"lengths": T(3, dtype=I64, index=1)}),
    ("window must be 0", {"window": -1}),
    ("belong to an FP8 cache", {"value_scale": 2.0}),
    ("out must match", {"out": T(3, 8, 32)}),
    ("dtype mismatch: 'out'", {"out": T(3, 8, 64, dtype=F32)}),
    ("lse must be", {"lse": T(3, 4, dtype=F32)}),
    ("lse must be float32", {"lse": T(3, 8)}),
    ("workspace must have", {"workspace": None, "page_table": T(3, 400, dtype=I64)}),
    ("workspace must have", {"workspace": T(7, dtype=F32), "page_table": T(3, 400, dtype=I64)}),
])
def test_paged_attention_refuses(match, kw):
    raises(match, native.paged_attention_fwd, *attention_args(**kw))


def test_the_python_way_refuses_cpu_tensors():
    x, f = torch.zeros(5, 4, 64), torch.zeros(32, dtype=F64)
    p, cache, table = torch.zeros(5, dtype=I64), torch.zeros(3, 16, 4, 64), torch.zeros(5, 1, dtype=I64)
    for call in (lambda: K.rope_at(x, x, p, f), lambda: K.rope_at(x, x, p, f, inplace=True),
                 lambda: K.rope_to_cache(x, x, x, cache, cache, p, p, f),
                 lambda: K.paged_attention(x, cache, cache, table, p)):
        with pytest.raises(ValueError, match="must be a CUDA tensor, got device type 'cpu'"):
            call()


def test_native_calls_leave_other_arguments_to_the_long_way():
    x, f, p = torch.zeros(5, 4, 64), torch.zeros(32, dtype=F64), torch.zeros(5, dtype=I64)
    cache, table = torch.zeros(3, 16, 4, 64), torch.zeros(5, 1, dtype=I64)
    calls = {"rope_at_call": (x, x, p, f, "half", 1.0, False, False),
             "rope_to_cache_call": (x, x, x, cache, cache, p, p, f, "half", 1.0, 1.0, 1.0, False),
             "paged_attention_call": (x, cache, cache, table, p, 0.1, 0, 1.0, 1.0, False)}
    for name, args in calls.items():
        call = getattr(native, name)
        assert call(*args) is None and call() is None and call(*args, None) is None
        for i in range(len(args)):
            for other in (None, object(), 3, 2.5, "e4m3", 1 << 80, [1], x.numpy()):
                assert call(*args[:i], other, *args[i + 1:]) is None


def test_frequencies():
    f, scale = K.rope_frequencies(8, 10000.0, device="cpu")
    assert f.dtype == F64 and scale == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=F64), rtol=1e-15)
    assert K.rope_frequencies(0, device="cpu")[0].shape == (0,)
    linear, _ = K.rope_frequencies(8, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(linear, f / 4)
    ntk, _ = K.rope_frequencies(8, scaling="ntk", factor=4.0, device="cpu")
    # the fastest pair stays, the slowest is divided by the factor
    assert ntk[0] == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    for kind, high, want in (("parts", 4.0, 1.0), ("yarn", 32.0, 0.1 * math.log(4.0) + 1.0)):
        g, scale = K.rope_frequencies(64, scaling=kind, factor=4.0, original_length=1000, device="cpu")
        plain, _ = K.rope_frequencies(64, device="cpu")
        turns = 1000 * plain / (2 * math.pi)
        assert scale == want
        assert torch.equal(g[turns >= high], plain[turns >= high])
        assert torch.equal(g[turns <= 1.0], plain[turns <= 1.0] / 4)
        between = (turns > 1.0) & (turns < high)
        share = (turns[between] - 1) / (high - 1)
        assert torch.allclose(g[between], plain[between] * (share + (1 - share) / 4), rtol=1e-12)
    for bad in ({"rotary_dim": 7}, {"rotary_dim": -2}, {"rotary_dim": 8, "scaling": "dynamic"},
                {"rotary_dim": 8, "theta": 0.0}, {"rotary_dim": 8, "factor": 0.5}, {"rotary_dim": 8, "theta": math.nan},
                {"rotary_dim": 8, "scaling": "parts", "low": 4.0, "high": 4.0}):
        with pytest.raises(ValueError):
            K.rope_frequencies(**{"device": "cpu", **bad})


def test_oracle_attention_and_rotation_against_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, generator=g, dtype=F64) for n in ((2, 4, 8), (10, 2, 8), (10, 2, 8)))
    keys, values = k.view(5, 2, 2, 8), v.view(5, 2, 2, 8)
    table = torch.arange(5).expand(2, 5)
    out, lse, _, _ = decode.paged_attention(q.numpy(), keys.numpy(), values.numpy(), table.numpy(), np.array([10, 7]))
    for b, n in ((0, 10), (1, 7)):
        kk, vv = (t[:n].repeat_interleave(2, 1).transpose(0, 1) for t in (k, v))
        s = (kk @ q[b].unsqueeze(-1)).squeeze(-1) / math.sqrt(8)
        assert torch.allclose(torch.from_numpy(lse[b]), s.logsumexp(-1))
        assert torch.allclose(torch.from_numpy(out[b]), (s.softmax(-1).unsqueeze(1) @ vv).squeeze(1))
    x = torch.randn(3, 2, 6, generator=g, dtype=F64)
    turned = decode.rope_at(x.numpy(), [0, 1, 2], [0.5, 0.25], "interleaved", 2.0)
    z = torch.view_as_complex(x[..., :4].reshape(3, 2, 2, 2)) * torch.polar(
        torch.full((3, 1, 2), 2.0, dtype=F64), torch.arange(3.0, dtype=F64)[:, None, None] * torch.tensor([0.5, 0.25]))
    assert np.allclose(turned[..., :4], torch.view_as_real(z).flatten(-2).numpy()) and np.array_equal(
        turned[..., 4:], x[..., 4:].numpy())


def test_the_planted_mistake_is_seen():
    """The bounds of the GPU tests tell a rotation by a neighbouring position apart."""
    x = np.random.default_rng(0).standard_normal((4, 2, 64))
    f = K.rope_frequencies(64, device="cpu")[0].numpy()
    a, b = decode.rope_at(x, [5, 6, 7, 8], f), decode.rope_at(x, [5, 6, 7, 9], f)
    off = np.abs(a - b)[3]
    assert (off > 2.0 ** -21 * 2 * np.abs(x).max() + 2.0 ** -8).any() and np.array_equal(a[:3], b[:3])
    assert ofp8.FP8_MAX["e4m3"] == 448.0


def linear_args(**kw):
    a = {"x": T(5, 300, dtype=E4M3), "xs": T(5, 3, dtype=F32), "w": T(200, 300, dtype=E4M3), "ws": T(2, 3, dtype=F32),
         "offsets": None, "y": T(5, 200)}
    return [{**a, **kw}[n] for n in a]


GROUPED = {"w": T(4, 200, 300, dtype=E4M3), "ws": T(4, 2, 3, dtype=F32), "offsets": T(5, dtype=I64)}


@pytest.mark.parametrize("match,kw", [
    ("x_codes must be float8", {"x": T(5, 300)}),
    ("w_codes must be float8", {"w": T(200, 300, dtype=F32)}),
    ("x_scale must be float32", {"xs": T(5, 3)}),
    ("w_scale must be float32", {"ws": T(2, 3)}),
    ("unsupported dtype", {"y": T(5, 200, dtype=E4M3)}),
    ("device mismatch: 'w_codes'", {"w": T(200, 300, dtype=E4M3, index=1)}),
    ("must be contiguous", {"w": T(200, 300, dtype=E4M3, strides=(1, 200))}),
    ("x_codes must be 2-D", {"x": T(1, 5, 300, dtype=E4M3)}),
    ("w_codes must be", {"w": T(200, 301, dtype=E4M3)}),
    ("w_codes must be", {"w": T(4, 200, 300, dtype=E4M3)}),
    ("w_codes must be", {**GROUPED, "w": T(3, 200, 300, dtype=E4M3)}),
    ("offsets must be int64", {**GROUPED, "offsets": T(5, dtype=torch.int32)}),
    ("num_experts in", {**GROUPED, "offsets": T(1, dtype=I64)}),
    ("x_scale shape", {"xs": T(5, 2, dtype=F32)}),
    ("x_scale shape", {"xs": T(3, 3, dtype=F32)}),
    ("w_scale shape", {"ws": T(200, 3, dtype=F32)}),
    ("w_scale shape", {**GROUPED, "ws": T(2, 3, dtype=F32)}),
    ("y shape", {"y": T(5, 201)}),
    ("4 MiB", {"x": T(5, 1 << 23, dtype=E4M3), "xs": T(5, 1 << 16, dtype=F32), "w": T(200, 1 << 23, dtype=E4M3),
               "ws": T(2, 1 << 16, dtype=F32)}),
])
def test_fp8_block_linear_refuses(match, kw):
    raises(match, native.fp8_block_linear_fwd, *linear_args(**kw))


def test_group_quant_refuses():
    for match, args in (("scale shape", (T(5, 300), T(5, 300, dtype=E4M3), T(5, 2, dtype=F32), "e4m3")),
                        ("x_fp8 shape", (T(5, 300), T(5, 299, dtype=E4M3), T(5, 3, dtype=F32), "e4m3")),
                        ("x must be 2-D", (T(300), T(300, dtype=E4M3), T(3, dtype=F32), "e4m3")),
                        ("fp8_format", (T(5, 300), T(5, 300, dtype=E4M3), T(5, 3, dtype=F32), "e3m4"))):
        raises(match, native.fp8_quant_group_fwd, *args)
    raises("static scale is per-tensor", K.fp8_quant, torch.zeros(2, 128), "e4m3", "group", 0.5)
    raises("must be a CUDA tensor", K.fp8_quant, torch.zeros(2, 128), "e4m3", "group")


def test_the_python_linear_refuses_cpu_tensors():
    x, w = torch.zeros(5, 128).to(E4M3), torch.zeros(7, 128).to(E4M3)
    raises("must be a CUDA tensor", K.fp8_block_linear, x, torch.ones(5, 1), w, torch.ones(1, 1))
    raises("x_codes must be 2-D", K.fp8_block_linear, x[0], torch.ones(1), w, torch.ones(1, 1))
    raises("w_codes 3-D", K.fp8_block_linear, x, torch.ones(5, 1), w, torch.ones(1, 1), torch.zeros(2, dtype=I64))
    args = (x, torch.ones(5, 1), w, torch.ones(1, 1), None, BF16)
    for i in range(len(args)):
        for other in (None, object(), 3, 2.5, "e4m3", 1 << 80, [1]):
            assert native.fp8_block_linear_call(*args[:i], other, *args[i + 1:]) is None


def test_launchers_refuse_and_take_nothing():
    """Through the C ABI: 0 for no work, hipErrorInvalidValue (1) for sizes, tags and scales out of range,
    both before any device call."""
    import ctypes

    from tests import _cck

    lib, p, strides = _cck.load(), 1 << 20, (ctypes.c_int64 * 8)(*[64] * 8)
    s = ctypes.cast(strides, ctypes.c_void_p)

    def rope(tokens=1, dim=64, half=32, dtype=2):
        return lib.launch_rope_at_fwd(p, p, p, p, p, p, s, tokens, 1, 1, dim, half, 0, 0, 1.0, dtype, None)

    assert rope(tokens=0) == 0 and rope(dim=0) == 0
    assert rope(dtype=3) == 1 and rope(half=33) == 1 and rope(half=-1) == 1 and rope(dim=4096) == 1

    def cache(tokens=1, key_scale=1.0, cache_dtype=3, half=32):
        return lib.launch_rope_to_cache_fwd(p, p, p, p, p, p, p, p, p, s, tokens, 1, 1, 64, half, 16, 0, 1.0, key_scale,
                                            1.0, 2, cache_dtype, None)

    assert cache(tokens=0) == 0
    assert cache(key_scale=0.0) == 1 and cache(key_scale=math.inf) == 1 and cache(cache_dtype=1) == 1 and cache(half=40) == 1

    def attention(sequences=1, heads=8, kv=2, dim=64, page=16, width=2, dtype=2, cache_dtype=2, workspace=None):
        return lib.launch_paged_attention_fwd(p, p, p, p, p, p, None, workspace, 512, 64, sequences, heads, kv, dim, 9, page,
                                              width, 0, 1.0, 1.0, 1.0, dtype, cache_dtype, None)

    assert attention(sequences=0) == 0 and attention(heads=0) == 0
    for bad in ({"heads": 7}, {"kv": 0}, {"dim": 72}, {"dim": 272}, {"page": 0}, {"width": -1}, {"width": 1 << 27},
                {"dtype": 3}, {"cache_dtype": 1}, {"width": 400}, {"width": 400, "workspace": p + 4},
                {"sequences": 1 << 23}):
        assert attention(**bad) == 1, bad
    room = lib.cck_paged_attention_workspace
    room.restype, room.argtypes = ctypes.c_int64, [ctypes.c_int64] * 6 + [ctypes.c_int32]
    assert room(1, 8, 2, 64, 16, 2, 2) == 0 and room(1, 8, 2, 64, 16, 400, 3) > 0 and room(1, 7, 2, 64, 16, 400, 2) == 0

    def linear(rows=1, experts=1, n=16, k=128, block_rows=1, fx=3, fw=3, dtype=2):
        return lib.launch_fp8_block_linear_fwd(p, p, p, p, None, p, rows, experts, n, k, block_rows, fx, fw, dtype, None)

    assert linear(rows=0) == 0 and linear(n=0) == 0
    for bad in ({"experts": 2}, {"block_rows": 64}, {"fx": 2}, {"fw": 0}, {"dtype": 3}, {"k": 1 << 23}, {"rows": 1 << 31}):
        assert linear(**bad) == 1, bad
    assert lib.launch_fp8_quant_group_fwd(p, p, p, 0, 5, 2, 3, None) == 0
    assert lib.launch_fp8_quant_group_fwd(p, p, p, 1, 1 << 31, 2, 3, None) == 1
    assert lib.launch_fp8_quant_group_fwd(p, p, p, 1, 5, 2, 2, None) == 1
