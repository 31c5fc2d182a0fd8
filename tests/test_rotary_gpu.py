"""rope_at and rope_to_cache against the float64 formulas of oracle/decode.py.

Bounds. Sine and cosine: the angle's rest is rounded to float32 below pi / 4 (2^-25),
the series and their five steps are off by less than 2^-23, the factor rounds once more
(2^-24): together less than 2^-22 of the factor. Each result is two products and a sum,
rounded to at most 2^-23 of factor (|a| + |b|). So 2^-21 factor (|a| + |b|), and the
output's own rounding, eps / 2 of the value (half the smallest subnormal at least).
An FP8 code is the nearest value to a quotient that is off by that and by its own
rounding, so it is off by half a step at most, and by the quotient's error beyond.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from oracle import decode
from oracle import fp8 as ofp8

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = [str(d).split(".")[-1] for d in DTYPES]
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


def _rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _positions(shape, most, seed):
    return torch.randint(0, most, shape, generator=torch.Generator().manual_seed(seed))


def _pair_sum(x, half, layout):
    """|a| + |b| of each element's pair, 0 for elements that are copied."""
    x = np.abs(x)
    out = np.zeros_like(x)
    first = slice(0, half) if layout == "half" else slice(0, 2 * half, 2)
    second = slice(half, 2 * half) if layout == "half" else slice(1, 2 * half, 2)
    out[..., first] = out[..., second] = x[..., first] + x[..., second]
    return out


def _bound(x, want, half, layout, factor, dtype):
    info = torch.finfo(dtype)
    own = np.maximum(np.abs(want) * info.eps / 2, info.smallest_normal * info.eps / 2)
    return abs(factor) * 2.0 ** -21 * _pair_sum(x, half, layout) + own


def _check(got, x, positions, frequencies, layout, factor, inverse, dtype):
    x64 = x.double().numpy()
    want = decode.rope_at(x64, positions.numpy(), frequencies.cpu().numpy(), layout, factor, inverse)
    off = np.abs(got.double().cpu().numpy() - want)
    bound = _bound(x64, want, len(frequencies), layout, factor, dtype)
    assert got.dtype == dtype and got.shape == x.shape
    assert (off <= bound).all(), (off / bound).max()
    rest = 2 * len(frequencies)
    assert torch.equal(got.cpu()[..., rest:], x[..., rest:])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary", [
    (1, 1, 1, 2, 2), (1, 32, 8, 128, 128), (5, 4, 4, 64, 32), (33, 3, 1, 80, 52), (7, 2, 2, 75, 30), (3, 5, 2, 9, 0),
    (300, 2, 1, 24, 24), (17, 6, 3, 256, 256), (2000, 1, 1, 16, 6), (2, 1, 3, 2048, 2048), (1300, 9, 2, 36, 36)])
def test_against_float64(tokens, heads, kv, dim, rotary, layout, dtype):
    frequencies, factor = K.rope_frequencies(rotary, 500000.0, scaling="yarn", factor=4.0)
    q, k = _rand((tokens, heads, dim), dtype, 1), _rand((tokens, kv, dim), dtype, 2)
    positions = _positions((tokens,), 1 << 17, 3)
    for inverse in (False, True):
        out = K.rope_at(q.cuda(), k.cuda(), positions.cuda(), frequencies, layout=layout, scale=factor,
                        inverse=inverse)
        for got, x in zip(out, (q, k)):
            _check(got, x, positions, frequencies, layout, factor, inverse, dtype)
    qd, kd = q.cuda(), k.cuda()
    got = K.rope_at(qd, kd, positions.cuda(), frequencies, layout=layout, scale=factor, inverse=True, inplace=True)
    assert got[0] is qd and got[1] is kd and torch.equal(qd, out[0]) and torch.equal(kd, out[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_far_and_negative_positions(dtype):
    positions = torch.tensor([0, 1, -1, 100003, -99999, (1 << 24) + 1, (1 << 31) - 1, -(1 << 31)])
    frequencies, _ = K.rope_frequencies(64)
    x = _rand((8, 2, 64), dtype, 5)
    # float64 holds the angle 2^31 to 2^-22; the reference's has the same error.
    for got in K.rope_at(x.cuda(), x.clone().cuda(), positions.cuda(), frequencies):
        x64 = x.double().numpy()
        want = decode.rope_at(x64, positions.numpy(), frequencies.cpu().numpy())
        angle = np.abs(positions.numpy())[:, None, None] * 2.0 ** -51
        bound = _bound(x64, want, 32, "half", 1.0, dtype) + angle * _pair_sum(x64, 32, "half")
        assert (np.abs(got.double().cpu().numpy() - want) <= bound).all()


def test_strided_heads_and_leading_dimensions():
    """Slices of one projection's output, in place and out of it; [B, S, H, D]."""
    frequencies, _ = K.rope_frequencies(64)
    qkv = _rand((37, (6 + 2 + 2) * 64), torch.bfloat16, 7).cuda()
    q, k = qkv[:, :6 * 64].unflatten(1, (6, 64)), qkv[:, 6 * 64:8 * 64].unflatten(1, (2, 64))
    positions = _positions((37,), 5000, 8).cuda()
    want = K.rope_at(q.contiguous(), k.contiguous(), positions, frequencies)
    got = K.rope_at(q, k, positions, frequencies)
    assert all(a.is_contiguous() and torch.equal(a, b) for a, b in zip(got, want))
    flipped = q.contiguous().transpose(0, 1).contiguous().transpose(0, 1)  # heads first in memory
    assert torch.equal(K.rope_at(flipped, k, positions, frequencies)[0], want[0])
    one = K.rope_at(q[:1].expand(37, 6, 64), k, positions, frequencies)[0]
    assert torch.equal(one, K.rope_at(q[:1].repeat(37, 1, 1), k, positions, frequencies)[0])
    v = qkv[:, 8 * 64:].clone()
    K.rope_at(q, k, positions, frequencies, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 8 * 64:], v)
    q4, k4 = _rand((3, 5, 4, 64), torch.float32, 9).cuda(), _rand((3, 5, 1, 64), torch.float32, 10).cuda()
    p4 = _positions((3, 5), 5000, 11).cuda()
    a = K.rope_at(q4, k4, p4, frequencies)
    b = K.rope_at(q4.flatten(0, 1), k4.flatten(0, 1), p4.flatten(), frequencies)
    assert all(torch.equal(x.flatten(0, 1), y) for x, y in zip(a, b))


@pytest.mark.parametrize("offset", [1, 3])
def test_unaligned(offset):
    frequencies, _ = K.rope_frequencies(64)
    flat = _rand((offset + 11 * 64,), torch.float16, 12).cuda()
    x, k, positions = flat[offset:].view(11, 1, 64), flat[offset:].view(11, 1, 64).clone(), _positions((11,), 99, 13)
    a = K.rope_at(x, k, positions.cuda(), frequencies)
    assert torch.equal(a[0], a[1])


def test_as_rope_on_its_positions():
    """rope's tables of 0 .. S - 1, whose angles are float32: as near as those are."""
    q, k = _rand((2, 64, 4, 128), torch.float32, 14).cuda(), _rand((2, 64, 2, 128), torch.float32, 15).cuda()
    frequencies, _ = K.rope_frequencies(128, 500000.0)
    angle = torch.arange(64, dtype=torch.float64, device="cuda")[:, None] * frequencies
    want = K.rope(q, k, angle.cos().float(), angle.sin().float())
    got = K.rope_at(q, k, torch.arange(64, device="cuda").expand(2, 64).contiguous(), frequencies)
    assert all((a - b).abs().max() < 2.0 ** -19 * 5 for a, b in zip(got, want))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_gradient(layout):
    """<g, R x> = <R^T g, x>, R^T by the formula's gradient and by differences (R is linear, so exact ones)."""
    frequencies, factor = K.rope_frequencies(40, scaling="yarn", factor=8.0)
    x, g = _rand((9, 3, 48), torch.float32, 16), _rand((9, 3, 48), torch.float32, 17)
    positions = _positions((9,), 3000, 18)
    grad = K.rope_at(g.cuda(), g.clone().cuda(), positions.cuda(), frequencies, layout=layout, scale=factor,
                     inverse=True)[0].double().cpu()
    leaf = x.double().requires_grad_()
    half = 20
    angle = positions.double()[:, None, None] * frequencies.cpu()
    c, s = factor * angle.cos(), factor * angle.sin()
    a, b = (leaf[..., :half], leaf[..., half:40]) if layout == "half" else (leaf[..., 0:40:2], leaf[..., 1:40:2])
    turned = torch.cat([a * c - b * s, b * c + a * s, leaf[..., 40:]], -1)
    order = torch.cat([g[..., :40], g[..., 40:]], -1) if layout == "half" else torch.cat(
        [g[..., 0:40:2], g[..., 1:40:2], g[..., 40:]], -1)
    (turned * order.double()).sum().backward()
    bound = 2.0 ** -21 * factor * _pair_sum(g.numpy(), half, layout) + 2.0 ** -24 * leaf.grad.abs().numpy()
    assert (np.abs(grad.numpy() - leaf.grad.numpy()) <= bound).all()
    step = torch.zeros_like(x)
    step[4, 1, 5] = 1.0
    up = K.rope_at((x + step).cuda(), x.cuda(), positions.cuda(), frequencies, layout=layout, scale=factor)
    difference = ((up[0] - up[1]).double().cpu() * g.double()).sum()
    # both sides of the difference are rounded: a dozen float32 roundings of values below 8
    assert abs(float(difference - grad[4, 1, 5])) < 2.0 ** -16


def test_infinities_stay_in_their_pairs():
    frequencies, _ = K.rope_frequencies(16)
    x = _rand((4, 2, 24), torch.float32, 19)
    x[1, 0, 3], x[2, 1, 20] = float("inf"), float("nan")
    got = K.rope_at(x.cuda(), x.clone().cuda(), torch.arange(1, 5).cuda(), frequencies)[0].cpu()
    bad = ~got.isfinite()
    want = torch.zeros_like(bad)
    want[1, 0, 3] = want[1, 0, 11] = want[2, 1, 20] = True
    assert torch.equal(bad, want)


def test_no_tokens_no_heads():
    frequencies, _ = K.rope_frequencies(64)
    q, k = K.rope_at(torch.empty(0, 4, 64, device="cuda"), torch.empty(0, 2, 64, device="cuda"),
                     torch.empty(0, dtype=torch.int64, device="cuda"), frequencies)
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    x, positions = _rand((3, 4, 64), torch.float32, 20).cuda(), torch.arange(3, device="cuda")
    q, k = K.rope_at(x, x[:, :0], positions, frequencies)
    assert k.shape == (3, 0, 64) and torch.equal(q, K.rope_at(x, x.clone(), positions, frequencies)[1])


# ---------------------------------------------------------------------------
# rope_to_cache
# ---------------------------------------------------------------------------

def _check_codes(codes, fmt, want, error):
    """FP8 codes of values `want` that are known to `error`."""
    most = ofp8.FP8_MAX[fmt]
    want = np.clip(want, -most, most)
    got = ofp8.decode(codes, fmt).astype(np.float64)
    mantissa, lowest = (3, -6) if fmt == "e4m3" else (2, -14)
    # half a step at the larger of the two: a value near a power of two may round to it from both sides
    power = np.floor(np.log2(np.maximum(np.maximum(np.abs(want), np.abs(got)), 2.0 ** lowest)))
    assert (np.abs(got - want) <= 2.0 ** (power - mantissa - 1) + error).all()
    assert (np.abs(got) <= most).all()


@pytest.mark.parametrize("cache", ["same", "e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("tokens,heads,kv,dim,rotary,layout", [
    (1, 32, 8, 128, 128, "half"), (16, 4, 4, 80, 52, "interleaved"), (33, 3, 1, 75, 30, "half"),
    (700, 8, 2, 64, 64, "interleaved"), (9, 2, 1, 48, 0, "half"), (1200, 4, 1, 32, 32, "half")])
def test_to_cache(tokens, heads, kv, dim, rotary, layout, dtype, cache):
    frequencies, factor = K.rope_frequencies(rotary, scaling="yarn", factor=2.0)
    q, k, v = (_rand((tokens, n, dim), dtype, 30 + n) for n in (heads, kv, kv))
    k[0, 0, :4] = 1000.0  # past e4m3's largest
    positions, page = _positions((tokens,), 9000, 31), 7
    pages = tokens // page + 3
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(32))[:tokens]
    slots[tokens // 2] = -1 if tokens % 2 else pages * page
    kept = torch.tensor([i for i in range(tokens) if 0 <= slots[i] < pages * page], dtype=torch.int64)
    cache_type = dtype if cache == "same" else FP8[cache]
    fill = torch.full((pages, page, kv, dim), 3.0).to(cache_type).cuda()
    keys, values = fill.clone(), fill.clone()
    ks, vs = (1.0, 1.0) if cache == "same" else (0.37, 0.011)
    got = K.rope_to_cache(q.cuda(), k.cuda(), v.cuda(), keys, values, slots.cuda(), positions.cuda(), frequencies,
                          layout=layout, scale=factor, key_scale=ks, value_scale=vs)
    _check(got, q, positions, frequencies, layout, factor, False, dtype)
    written = np.zeros(pages * page, dtype=bool)
    written[slots[kept].numpy()] = True
    raw = torch.uint8 if cache != "same" else cache_type
    for out, x, scale, turned in ((keys, k, ks, True), (values, v, vs, False)):
        rows = out.view(raw).cpu().flatten(0, 1)
        assert torch.equal(rows[~written], fill.view(raw).cpu().flatten(0, 1)[~written])  # the others as they were
        rows, x = rows[slots[kept]], x[kept]
        if cache == "same":
            if turned:
                _check(rows, x, positions[kept], frequencies, layout, factor, False, dtype)
            else:
                assert torch.equal(rows, x)
            continue
        x64, scale32 = x.double().numpy(), float(np.float32(scale))
        want, error = x64, np.zeros(x64.shape)
        if turned:
            want = decode.rope_at(x64, positions[kept].numpy(), frequencies.cpu().numpy(), layout, factor)
            error = factor * 2.0 ** -21 * _pair_sum(x64, rotary // 2, layout)
        _check_codes(rows.numpy(), cache, want / scale32, (error + np.abs(want) * 2.0 ** -24) / scale32)
    same = q.cuda()
    again = K.rope_to_cache(same, k.cuda(), v.cuda(), keys, values, slots.cuda(), positions.cuda(), frequencies,
                            layout=layout, scale=factor, key_scale=ks, value_scale=vs, inplace=True)
    assert again is same and torch.equal(same, got)


def test_to_fp8_cache_is_exact_where_the_quotient_is():
    """Values (not turned) by a power of two: the codes of the nearest value, ties to even, NaN and infinities."""
    x = torch.arange(0, 65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    v = x.reshape(512, 1, 128)
    k, slots = torch.zeros_like(v), torch.arange(512)
    for fmt, cache in FP8.items():
        keys = torch.zeros(512, 1, 1, 128, device="cuda").to(cache)
        values = keys.clone()
        K.rope_to_cache(k.cuda(), k.cuda(), v.cuda(), keys, values, slots.cuda(), slots.cuda(),
                        torch.empty(0, dtype=torch.float64, device="cuda"), key_scale=0.5, value_scale=0.5)
        most = ofp8.FP8_MAX[fmt]
        want = ofp8.encode(np.clip(x.float().numpy() / np.float32(0.5), -most, most), fmt)
        got = values.view(torch.uint8).cpu().numpy().ravel()
        nan = x.isnan().numpy()
        assert np.array_equal(got[~nan], want[~nan])
        assert np.isnan(ofp8.decode(got[nan], fmt)).all()


def test_cache_of_strided_slices():
    frequencies, _ = K.rope_frequencies(64)
    qkv = _rand((21, 8 * 64), torch.bfloat16, 40).cuda()
    q, k, v = (qkv[:, a * 64:b * 64].unflatten(1, (b - a, 64)) for a, b in ((0, 4), (4, 6), (6, 8)))
    slots, positions = torch.randperm(32)[:21].cuda(), _positions((21,), 999, 41).cuda()
    caches = [torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    want = K.rope_to_cache(q.contiguous(), k.contiguous(), v.contiguous(), *caches[:2], slots, positions, frequencies)
    got = K.rope_to_cache(q, k, v, *caches[2:], slots, positions, frequencies, inplace=True)
    assert torch.equal(got, want) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])


# ---------------------------------------------------------------------------
# Many tokens: the same bits as of small calls.
# ---------------------------------------------------------------------------

def _in_chunks(fn, count, *tensors):
    parts = [fn(*(t[i:i + count] for t in tensors)) for i in range(0, len(tensors[0]), count)]
    return [torch.cat(p) for p in zip(*parts)]


LARGE = [(torch.bfloat16, 4099, 56, 8, 128, 128, "half"), (torch.bfloat16, 4099, 56, 8, 128, 128, "interleaved"),
         (torch.float32, 3001, 24, 24, 128, 64, "half"), (torch.float16, 16385, 32, 1, 64, 64, "interleaved")]


@pytest.mark.parametrize("dtype,tokens,heads,kv,dim,rotary,layout", LARGE)
def test_large(dtype, tokens, heads, kv, dim, rotary, layout):
    frequencies, _ = K.rope_frequencies(rotary, 500000.0)
    g = torch.Generator("cuda").manual_seed(50)
    q, k = (torch.randn((tokens, n, dim), generator=g, device="cuda").to(dtype) for n in (heads, kv))
    positions = _positions((tokens,), 1 << 20, 51).cuda()
    for inverse in (False, True):
        def rope(q, k, p, **how):
            return K.rope_at(q, k, p, frequencies, layout=layout, scale=1.25, inverse=inverse, **how)
        want = _in_chunks(rope, 500, q, k, positions)
        assert all(torch.equal(a, b) for a, b in zip(rope(q, k, positions), want))
    wide = torch.full((tokens, heads + kv + 3, dim), 2.0, dtype=dtype, device="cuda")
    wide[:, :heads], wide[:, heads:heads + kv] = q, k
    rope(wide[:, :heads], wide[:, heads:heads + kv], positions, inplace=True)
    assert torch.equal(wide[:, :heads], want[0]) and torch.equal(wide[:, heads:heads + kv], want[1])
    assert (wide[:, heads + kv:] == 2.0).all()


@pytest.mark.parametrize("cache", ["same", "e4m3", "e5m2"])
@pytest.mark.parametrize("dtype,tokens,heads,kv,dim,rotary,layout", LARGE[:3])
def test_large_to_cache(dtype, tokens, heads, kv, dim, rotary, layout, cache):
    frequencies, _ = K.rope_frequencies(rotary, 500000.0)
    g = torch.Generator("cuda").manual_seed(52)
    q, k, v = (torch.randn((tokens, n, dim), generator=g, device="cuda").to(dtype) for n in (heads, kv, kv))
    positions, page = _positions((tokens,), 1 << 20, 53).cuda(), 7
    pages = tokens // page + 3
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(54))[:tokens].cuda()
    slots[[5, tokens - 1]] = torch.tensor([-1, pages * page], device="cuda")
    kind = dtype if cache == "same" else FP8[cache]
    raw = dtype if cache == "same" else torch.uint8
    caches = [torch.full((pages, page, kv, dim), 3.0, device="cuda").to(kind) for _ in range(4)]
    scales = {} if cache == "same" else {"key_scale": 0.02, "value_scale": 0.3}

    def rope(keys, values, inplace=False):
        return lambda q, k, v, s, p: [K.rope_to_cache(q, k, v, keys, values, s, p, frequencies, layout=layout,
                                                      inplace=inplace, **scales)]
    want, = _in_chunks(rope(*caches[:2]), 500, q, k, v, slots, positions)
    assert torch.equal(rope(*caches[2:])(q, k, v, slots, positions)[0], want)
    assert all(torch.equal(caches[i].view(raw), caches[i + 2].view(raw)) for i in (0, 1))
    for c in caches[2:]:
        c.view(raw).zero_()
    same, = rope(*caches[2:], inplace=True)(q, k, v, slots, positions)
    assert same is q and torch.equal(q, want)
    written = slots[(slots >= 0) & (slots < pages * page)]
    assert all(torch.equal(caches[i].view(raw).flatten(0, 1)[written], caches[i + 2].view(raw).flatten(0, 1)[written])
               for i in (0, 1))


def test_more_tokens_than_workgroups():
    frequencies, _ = K.rope_frequencies(6)
    tokens = (1 << 21) + 5
    g = torch.Generator("cuda").manual_seed(55)
    q = torch.randn((tokens, 1, 6), generator=g, device="cuda").half()
    positions = torch.randint(0, 1 << 17, (tokens,), generator=g, device="cuda")
    want = _in_chunks(lambda q, p: K.rope_at(q, q[:, :0], p, frequencies), 1 << 20, q, positions)[0]
    assert torch.equal(K.rope_at(q, q[:, :0], positions, frequencies)[0], want)
