"""paged_attention against the float64 formula of oracle/decode.py.

Bounds. A score is a float32 sum of D products (16-bit and FP8 ones exact), so it is off by
at most (D + 4) 2^-24 of the sum of |scale q k|, scaling included; call that d (it is a
relative error of p, of their sum and so of the output 2 d, and an absolute one of lse).
The exponentials, their sums over L positions in any order and the joins of parts add
(L + 64) 2^-24 at most, in practice the square root of it; 16-bit P in two parts adds 2^-16
(bfloat16) or 2^-21. An FP8 cache's scale is float32 (2^-24). So the output is off by
(2 d + 2^-16 + (2 L + 128) 2^-24) sum p |v| and its own rounding.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from oracle import decode

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = [str(d).split(".")[-1] for d in DTYPES]
U = 2.0 ** -24


def _case(lengths, heads, kv, dim, page, dtype, cache=None, seed=0, spare=2):
    g = torch.Generator().manual_seed(seed)
    b, cache = len(lengths), cache or dtype
    per = max(1, -(-max(lengths) // page))
    pages = b * per + spare
    q = (torch.randn((b, heads, dim), generator=g) * 1.5).to(dtype)
    keys, values = (torch.randn((pages, page, kv, dim), generator=g).to(cache) for _ in range(2))
    table = torch.randperm(pages, generator=g)[:b * per].view(b, per)
    return q, keys, values, table, torch.tensor(lengths, dtype=torch.int64)


def _check(q, keys, values, table, lengths, got=None, **kw):
    scales = {n: kw.get(n, 1.0) for n in ("key_scale", "value_scale")}
    if got is None:
        got = K.paged_attention(q.cuda(), keys.cuda(), values.cuda(), table.cuda(), lengths.cuda(), return_lse=True, **kw)
    out, lse = got
    k64, v64 = (c.double().numpy() * float(np.float32(s)) for c, s in zip((keys, values), scales.values()))
    want, want_lse, spread, size = decode.paged_attention(q.double().numpy(), k64, v64, table.numpy(), lengths.numpy(),
                                                          kw.get("scale"), kw.get("window", 0))
    assert out.dtype == q.dtype and out.shape == q.shape and lse.dtype == torch.float32
    longest = max(1, int(lengths.max())) if len(lengths) else 1
    d = (q.shape[-1] + 4) * U * size
    info = torch.finfo(q.dtype)
    bound = ((2 * d + 2.0 ** -16 + (2 * longest + 128) * U)[..., None] * spread
             + np.maximum(np.abs(want) * info.eps / 2, info.smallest_normal * info.eps / 2))
    off = np.abs(out.double().cpu().numpy() - want)
    assert (off <= bound).all(), (off / np.maximum(bound, 1e-300)).max()
    lse = lse.double().cpu().numpy()
    assert np.array_equal(np.isinf(lse), np.isinf(want_lse))
    fine = ~np.isinf(want_lse)
    limit = d + (longest + 64) * U + np.abs(np.where(fine, want_lse, 0)) * 4 * U
    assert (np.abs(lse[fine] - want_lse[fine]) <= limit[fine]).all()
    return got


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 16), (8, 8, 64), (32, 8, 128), (12, 4, 80), (16, 1, 96), (14, 2, 192),
                                          (8, 2, 256), (40, 2, 64), (71, 1, 128), (3, 1, 48)])
def test_heads(heads, kv, dim, dtype):
    _check(*_case([0, 1, 17, 130, 333], heads, kv, dim, 16, dtype, seed=heads + dim))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("cache", [torch.float8_e4m3fn, torch.float8_e5m2], ids=["e4m3", "e5m2"])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (2, 2, 64), (12, 4, 80), (16, 1, 256)])
def test_fp8_cache(heads, kv, dim, cache, dtype):
    case = _case([5, 700, 129], heads, kv, dim, 16, dtype, cache, seed=dim)
    _check(*case, key_scale=0.31, value_scale=1.7)


@pytest.mark.parametrize("page", [1, 3, 7, 16, 13, 64, 100, 256, 4096])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_pages(page, dtype):
    _check(*_case([1, page, page + 1, 2 * page - 1, 515, 128, 129, 127], 8, 2, 64, page, dtype, seed=page))


@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 257, 511, 1025, 4095, 20000])
def test_one_sequence(length):
    _check(*_case([length], 8, 2, 128, 16, torch.bfloat16, seed=length))


def test_many_sequences():
    """More workgroups than parts are made for: one part each, no join."""
    g = torch.Generator().manual_seed(3)
    _check(*_case(torch.randint(0, 90, (700,), generator=g).tolist(), 8, 4, 64, 16, torch.bfloat16, seed=4))
    _check(*_case([64] * 3000, 2, 2, 32, 16, torch.float16, seed=5))


@pytest.mark.parametrize("window", [1, 5, 16, 100, 128, 129, 300, 100000])
def test_window(window):
    _check(*_case([0, 1, 99, 300, 301, 1000], 8, 2, 64, 16, torch.bfloat16, seed=window), window=window)


def test_absent_pages():
    """Pages outside the cache hold no positions; a sequence of them alone has none."""
    q, keys, values, table, lengths = _case([100, 400, 400, 64], 8, 2, 64, 16, torch.bfloat16, seed=6)
    pages = keys.shape[0]
    table[0, 2], table[1, 0], table[1, 5:9], table[3] = -1, pages, torch.tensor([-7, 1 << 40, pages + 3, -1]), -1
    table[2, ::2] = -1
    out, lse = _check(q, keys, values, table, lengths)
    assert (out[3] == 0).all() and torch.isinf(lse[3]).all() and (lse[3] < 0).all()
    none = keys[:0].cuda()
    out = K.paged_attention(q.cuda(), none, none, table.cuda(), lengths.cuda())
    assert (out == 0).all()


def test_lengths_past_the_table_and_below_nothing():
    q, keys, values, table, lengths = _case([160, 160, 160], 4, 2, 64, 16, torch.float32, seed=7)
    _check(q, keys, values, table, torch.tensor([-5, 1 << 40, 161]))
    _check(q, keys, values, table[:, :0], lengths)


def test_what_is_not_seen_may_hold_anything():
    """NaN and infinities behind the last position, before the window, and on other sequences' pages."""
    q, keys, values, table, lengths = _case([37, 200, 16], 8, 2, 128, 16, torch.bfloat16, seed=8)
    want = K.paged_attention(q.cuda(), keys.cuda(), values.cuda(), table.cuda(), lengths.cuda(), window=50)
    seen = torch.zeros(keys.shape[:2], dtype=torch.bool)
    for b in range(3):
        for t in range(max(0, int(lengths[b]) - 50), int(lengths[b])):
            seen[table[b, t // 16], t % 16] = True
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
        for target in (keys, values):
            target[~seen] = bad
        got = K.paged_attention(q.cuda(), keys.cuda(), values.cuda(), table.cuda(), lengths.cuda(), window=50)
        assert torch.equal(got, want), bad


def test_keys_of_minus_infinity_are_as_masked():
    q, keys, values, table, lengths = _case([100], 4, 1, 64, 16, torch.float32, seed=9)
    q = q.abs()
    want_keys = keys.clone()
    keys[table[0, 3]] = -float("inf")  # scores of -infinity
    got = K.paged_attention(q.cuda(), keys.cuda(), values.cuda(), table.cuda(), lengths.cuda(), return_lse=True)
    hidden = table.clone()
    hidden[0, 3] = -1
    _check(q, want_keys, values, hidden, lengths, got=got)


def test_a_score_of_nan_reaches_its_head_alone():
    q, keys, values, table, lengths = _case([300, 300], 4, 2, 64, 16, torch.bfloat16, seed=10)
    keys[table[1, 4], 3, 1, 7] = float("nan")
    out, lse = K.paged_attention(q.cuda(), keys.cuda(), values.cuda(), table.cuda(), lengths.cuda(), return_lse=True)
    nan = out.isnan().all(-1).cpu()
    assert nan.tolist() == [[False] * 4, [False, False, True, True]] and torch.equal(lse.isnan().cpu(), nan)
    assert not out[:, :2].isnan().any()


@pytest.mark.parametrize("scale", [0.0, 0.02, 30.0])
def test_scales_and_steep_scores(scale):
    """At 30 one position has nearly all the weight, and the running maximum climbs often."""
    _check(*_case([700, 300], 8, 2, 64, 16, torch.float32, seed=11), scale=scale)


def test_rising_scores():
    """Each position's score above the one before: the sums are scaled again and again."""
    q, keys, values, table, lengths = _case([600], 4, 1, 32, 16, torch.bfloat16, seed=12)
    q[:] = 1.0
    for t in range(600):
        keys[table[0, t // 16], t % 16] = t / 8.0
    _check(q, keys, values, table, lengths)


def test_strided_queries():
    q, keys, values, table, lengths = _case([50, 170], 8, 2, 64, 16, torch.bfloat16, seed=13)
    args = keys.cuda(), values.cuda(), table.cuda(), lengths.cuda()
    want = K.paged_attention(q.cuda(), *args)
    wide = torch.zeros(2, 12 * 64, dtype=torch.bfloat16, device="cuda")
    wide[:, :8 * 64] = q.flatten(1).cuda()
    assert torch.equal(K.paged_attention(wide[:, :8 * 64].unflatten(1, (8, 64)), *args), want)
    flipped = q.cuda().transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(K.paged_attention(flipped, *args), want)


def test_unaligned_cache():
    q, keys, values, table, lengths = _case([90], 4, 2, 64, 16, torch.float16, seed=14)
    flat = torch.zeros(keys.numel() + 1, dtype=torch.float16, device="cuda")
    flat[1:] = keys.cuda().flatten()
    off = flat[1:].view(keys.shape)
    args = values.cuda(), table.cuda(), lengths.cuda()
    assert torch.equal(K.paged_attention(q.cuda(), off, *args), K.paged_attention(q.cuda(), keys.cuda(), *args))


def test_shared_pages():
    """Sequences with a common beginning share its pages; a page twice in one table counts twice."""
    q, keys, values, table, lengths = _case([200, 200], 8, 2, 64, 16, torch.float32, seed=15)
    table[1, :6] = table[0, :6]
    table[0, 8] = table[0, 2]
    _check(q, keys, values, table, lengths)


def test_lse_joins_parts_of_a_context():
    q, keys, values, table, lengths = _case([640], 8, 2, 64, 16, torch.float32, seed=16)
    args = q.cuda(), keys.cuda(), values.cuda()
    whole, lse = K.paged_attention(*args, table.cuda(), lengths.cuda(), return_lse=True)
    a, la = K.paged_attention(*args, table[:, :13].contiguous().cuda(), torch.tensor([13 * 16]).cuda(), return_lse=True)
    b, lb = K.paged_attention(*args, table[:, 13:].contiguous().cuda(), torch.tensor([640 - 13 * 16]).cuda(),
                              return_lse=True)
    both = torch.logaddexp(la, lb)
    joined = a * (la - both).exp()[..., None] + b * (lb - both).exp()[..., None]
    assert (both - lse).abs().max() < 2.0 ** -18 and (joined - whole).abs().max() < 2.0 ** -18


def test_past_four_gigabytes():
    """A cache of 4.5 GB: pages at its end."""
    page, kv, dim = 256, 8, 128
    pages = (9 << 29) // (page * kv * dim * 2) + 1
    keys = torch.zeros(pages, page, kv, dim, dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    q, few_k, few_v, table, lengths = _case([700, 3], 16, kv, dim, page, torch.bfloat16, seed=17)
    n = few_k.shape[0]
    keys[-n:], values[-n:] = few_k.cuda(), few_v.cuda()
    got = K.paged_attention(q.cuda(), keys, values, (table + pages - n).cuda(), lengths.cuda())
    want = K.paged_attention(q.cuda(), few_k.cuda(), few_v.cuda(), table.cuda(), lengths.cuda())
    assert torch.equal(got, want)


def test_no_sequences():
    q, keys, values, table, lengths = _case([3], 8, 2, 64, 16, torch.float32, seed=18)
    out, lse = K.paged_attention(q[:0].cuda(), keys.cuda(), values.cuda(), table[:0].cuda(), lengths[:0].cuda(),
                                 return_lse=True)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)


def test_same_bits_every_time():
    case = [t.cuda() for t in _case([3000, 100, 777], 32, 8, 128, 16, torch.bfloat16, seed=19)]
    first = K.paged_attention(*case, return_lse=True)
    for _ in range(5):
        again = K.paged_attention(*case, return_lse=True)
        assert torch.equal(again[0], first[0]) and torch.equal(again[1], first[1])


@pytest.mark.parametrize("cache", [None, torch.float8_e4m3fn], ids=["same", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_small_probabilities(dtype, cache):
    """One position of probability almost 1 and 2^18 of 2^-26 of it, which float16 has not got: 2^-8 of the sum
    together. Values 1 and 2, so out is 1 + 2^-8 / (1 + 2^-8) and each small probability counts."""
    n = (1 << 18) + 1
    q = torch.full((1, 1, 16), 2.0, dtype=dtype)
    keys = torch.zeros((n, 1, 1, 16), dtype=dtype)
    values = torch.full((n, 1, 1, 16), 2.0, dtype=dtype)
    for at in (0, n // 2, n - 1):
        keys[:], values[:] = 0.0, 2.0
        keys[at], values[at] = 1.0, 1.0  # its score: 32 scale
        args = q, keys.to(cache or dtype), values.to(cache or dtype), torch.arange(n)[None], torch.tensor([n])
        out, lse = K.paged_attention(*(t.cuda() for t in args), scale=26 * np.log(2.0) / 32, return_lse=True)
        tail = 2.0 ** -26 * (n - 1)
        want = 1.0 + tail / (1.0 + tail)
        # The exponent 26 in float32 is a relative 2^-19 of the tail; its n terms' sum, in parts of no more than 2^13
        # and these of no more than 2^10, 2^-10 of it at most; as float16, lifted by 2^7, its terms are 2^-19 and off
        # by 2^-25 at most: 2^-6. So less than 2^-5 of the tail, 2^-13, and the output's rounding.
        assert (out.double().cpu() - want).abs().max() <= 2.0 ** -13 + want * torch.finfo(dtype).eps / 2
        # lse = 26 log 2 + log(1 + tail): those of the sum's errors, and float32's own of 18.02
        assert abs(float(lse.cpu()) - (26 * np.log(2.0) + np.log1p(tail))) <= 2.0 ** -13 + 18.1 * 2.0 ** -22


def test_most_heads():
    """2^23 query heads in all: too many workgroups for parts of the sequences."""
    b, heads = 2048, 4096
    g = torch.Generator("cuda").manual_seed(60)
    q = torch.randn((b, heads, 16), generator=g, device="cuda").half()
    keys, values = (torch.randn((3, 16, heads, 16), generator=g, device="cuda").half() for _ in range(2))
    table, lengths = torch.tensor([[2, 0, 1]]).repeat(b, 1), torch.arange(b) % 49
    out, lse = K.paged_attention(q, keys, values, table.cuda(), lengths.cuda(), return_lse=True)
    some = torch.tensor([0, 1, 48, 1000, b - 1])
    _check(q[some].cpu(), keys.cpu(), values.cpu(), table[some], lengths[some], got=(out[some], lse[some]))


# ---------------------------------------------------------------------------
# Who takes a sequence - a wave, a workgroup's waves, or parts of it are shared out - is chosen by how many positions
# the table has room for: the same sequences with wider tables.
# ---------------------------------------------------------------------------

def _wide(table, pages):
    return torch.cat([table, torch.full((table.shape[0], pages), -1)], 1)


@pytest.mark.parametrize("lengths", [[0, 1, 17, 130, 333], [2500, 31, 0, 1030]], ids=["short", "long"])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("heads,kv,dim,cache", [
    (8, 8, 64, None), (32, 8, 128, None), (12, 4, 80, None), (14, 2, 192, None), (8, 2, 256, None), (40, 2, 48, None),
    (8, 2, 128, torch.float8_e4m3fn), (12, 4, 80, torch.float8_e5m2), (16, 1, 256, torch.float8_e4m3fn),
    (4, 2, 16, torch.float8_e5m2)])
def test_ways(heads, kv, dim, cache, dtype, lengths):
    q, keys, values, table, lengths = _case(lengths, heads, kv, dim, 16, dtype, cache, seed=heads + dim)
    kw = {} if cache is None else {"key_scale": 0.31, "value_scale": 1.7}
    for pages in (0, 1, 30, 1000):
        _check(q, keys, values, _wide(table, pages), lengths, **kw)


@pytest.mark.parametrize("page", [1, 3, 13, 100, 256])
@pytest.mark.parametrize("window", [0, 5, 129, 900, 1500])
def test_windows_and_pages_of_long_sequences(page, window):
    q, keys, values, table, lengths = _case([1300, 0, 2100, 1, 899, 900, 901], 4, 2, 64, page, torch.float16, seed=page)
    table[2, 700 // page] = -1
    _check(q, keys, values, table, lengths, window=window)
    _check(q, keys, values, _wide(table, 4096 // page), lengths, window=window)


@pytest.mark.parametrize("pages", [0, 1000])
def test_what_is_not_seen_of_any_way(pages):
    q, keys, values, table, lengths = _case([37, 1200, 16], 8, 2, 128, 16, torch.bfloat16, seed=61)
    args = q.cuda(), keys.cuda(), values.cuda(), _wide(table, pages).cuda(), lengths.cuda()
    for window in (0, 50):
        want = K.paged_attention(*args, window=window)
        seen = torch.zeros(keys.shape[:2], dtype=torch.bool)
        for b in range(3):
            t = torch.arange(max(0, int(lengths[b]) - window) if window else 0, int(lengths[b]))
            seen[table[b, t // 16], t % 16] = True
        for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min):
            for target in (args[1], args[2]):
                target[~seen.cuda()] = bad
            assert torch.equal(K.paged_attention(*args, window=window), want), (bad, window)
        args = q.cuda(), keys.cuda(), values.cuda(), *args[3:]


@pytest.mark.parametrize("count,most", [(300, 40), (300, 200), (300, 700), (70, 200), (70, 1500), (2100, 300)])
def test_batches(count, most):
    g = torch.Generator().manual_seed(count + most)
    lengths = torch.randint(0, most + 1, (count,), generator=g).tolist()
    lengths[count // 2] = most
    _check(*_case(lengths, 4, 4, 32, 16, torch.bfloat16, seed=62))


@pytest.mark.parametrize("pages", [0, 1000])
def test_each_way_into_a_graph(pages):
    """Replayed with other lengths and queries, eager calls between."""
    q, keys, values, table, lengths = _case([400, 130, 0, 777], 8, 2, 128, 16, torch.bfloat16, seed=63)
    args = q.cuda(), keys.cuda(), values.cuda(), _wide(table, pages).cuda(), lengths.cuda()
    K.paged_attention(*args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = K.paged_attention(*args)
    for i in range(4):
        args[4].copy_(torch.tensor([400 - 99 * i, i, 130 * i, 777 // (i + 1)]))
        args[0].copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, K.paged_attention(*args)), i


@pytest.mark.parametrize("most", [700, 3000])
def test_more_sequences_than_are_cut(most):
    g = torch.Generator().manual_seed(64)
    q = torch.randn((2100, 2, 16), generator=g).half()
    keys, values = (torch.randn((200, 16, 1, 16), generator=g).half() for _ in range(2))
    table = torch.randint(0, 200, (2100, -(-most // 16)), generator=g)
    lengths = torch.randint(0, 100, (2100,), generator=g)
    lengths[::70] = torch.randint(0, most + 1, (30,), generator=g)
    lengths[[5, 2099]] = most
    _check(q, keys, values, table, lengths)
