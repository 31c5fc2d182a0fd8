"""Rotary calls whose outputs share memory with what other threads of the launch read or
write are refused: overlaps of the two caches, of q and k in place, of a cache and its
inputs. On the CPU, every call ending in its refusal before a launch. Where elements only
lie between each other's (slices of one projection), the check has to say so: against the
addresses themselves, one by one, in the oracle below."""

from __future__ import annotations

import itertools
import random

import pytest
import torch

from custom_cuda_kernals_amd._lib import native
from tests.test_decode_cpu import E4M3, I64, T, cache_args, raises, rope_args

MATCH = "are the same memory, or share some of it"
PLACE = 1 << 30


def _addresses(shape, strides, ptr, size=2):
    tokens, heads, dim = shape
    return {ptr + size * (t * strides[0] + h * strides[1]) + i
            for t in range(tokens) for h in range(heads) for i in range(size * dim)}


def _overlap(**kw):
    """Whether rope_at_fwd says that q_out and k_out overlap. A call that it finds fine is kept from its launch by
    a k, checked later, that begins inside q_out."""
    a = rope_args(**kw)
    a[1] = T(*a[1].shape, ptr=a[4]._ptr + 1)
    with pytest.raises(ValueError, match=MATCH) as e:
        native.rope_at_fwd(*a)
    return "'k_out'" in str(e.value)


def test_overlaps_are_those_of_the_addresses():
    rng = random.Random(0)
    found = [0, 0]
    for _ in range(4000):
        tokens, dim = rng.choice([1, 1, 2, 3, 5]), rng.choice([2, 4])
        views = []
        stride = rng.choice([0, 0, 1, 2])
        for heads in (rng.randint(1, 4), rng.randint(1, 4)):
            if rng.random() < 0.3:  # heads apart from each other by all tokens
                strides = (dim + rng.choice([0, 0, 1]), 0, 1)
                strides = (strides[0], tokens * strides[0] + rng.choice([0, 3]), 1)
            else:
                head = dim * rng.choice([1, 1, 2]) + rng.choice([0, 0, 1])
                strides = (head * heads + stride * 4, head, 1)
            views.append(((tokens, heads, dim), strides))
        if rng.random() < 0.7:  # one row for both
            row = max(v[1][0] for v in views) + rng.choice([0, 4, 9])
            if all(v[1][1] <= v[1][0] for v in views):
                views = [(shape, (row, *strides[1:])) for shape, strides in views]
        at = PLACE + 2 * rng.randint(-30, 30)
        (sq, tq), (sk, tk) = views
        want = bool(_addresses(sq, tq, PLACE) & _addresses(sk, tk, at))
        if tokens > 1 and tq[0] != tk[0]:
            lo, hi = (min(_addresses(s, t, p)) for s, t, p in ((sq, tq, PLACE), (sk, tk, at)))
            ends = [max(_addresses(s, t, p)) for s, t, p in ((sq, tq, PLACE), (sk, tk, at))]
            want = lo <= ends[1] and hi <= ends[0]  # strides that differ: by their ranges
        half = dim // 2
        got = _overlap(q=T(*sq, ptr=PLACE << 3), k=T(*sk), q_out=T(*sq, strides=tq, ptr=PLACE),
                       k_out=T(*sk, strides=tk, ptr=at), positions=T(tokens, dtype=I64),
                       frequencies=T(half, dtype=torch.float64))
        assert got == want, (views, at - PLACE)
        found[want] += 1
    assert min(found) > 500, found


def test_rope_at_in_place():
    def inplace(q, k):
        return rope_args(q=q, k=k, q_out=q, k_out=k)

    row = (8 * 64, 64, 1)
    q = T(5, 4, 64, strides=row, ptr=PLACE)
    raises(MATCH, native.rope_at_fwd, *inplace(q, T(5, 2, 64, strides=row, ptr=PLACE + 3 * 128)))
    raises(MATCH, native.rope_at_fwd, *inplace(q, T(5, 2, 64, strides=row, ptr=PLACE + 7 * 128)))  # into the next row
    raises(MATCH, native.rope_at_fwd, *inplace(q, q))
    raises(MATCH, native.rope_at_fwd, *inplace(T(5, 4, 64, ptr=PLACE), T(5, 2, 64, ptr=PLACE + 5 * 512 - 2)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_rope_to_cache(dtype):
    size = 2 if dtype == torch.bfloat16 else 1
    bytes_ = 3 * 16 * 2 * 64 * size

    def call(**kw):
        a = {"key_cache": T(3, 16, 2, 64, dtype=dtype, ptr=PLACE), "value_cache": T(3, 16, 2, 64, dtype=dtype, ptr=2 * PLACE)}
        return cache_args(**{**a, **kw})

    fwd = native.rope_to_cache_fwd
    for off in (0, 1, bytes_ - 1):
        raises(f"'key_cache' and 'value_cache' {MATCH}", fwd, *call(value_cache=T(3, 16, 2, 64, dtype=dtype, ptr=PLACE + off)))
        raises(f"'key_cache' and 'value_cache' {MATCH}", fwd, *call(key_cache=T(3, 16, 2, 64, dtype=dtype, ptr=2 * PLACE + off)))
    for name, place in itertools.product(("q", "k", "v"), (1, 2)):
        cache = {1: "key_cache", 2: "value_cache"}[place]
        heads = 4 if name == "q" else 2
        inside = T(5, heads, 64, strides=(2 * heads * 64, 64, 1), ptr=place * PLACE + bytes_ - 2)
        raises(f"'{cache}' and '{name}' {MATCH}", fwd, *call(**{name: inside}))
    raises(f"'key_cache' and 'q_out' {MATCH}", fwd, *call(q_out=T(5, 4, 64, ptr=PLACE - 2)))
    q = T(5, 4, 64, ptr=5 * PLACE)
    for name in ("k", "v"):
        raises(f"'q_out' and '{name}' {MATCH}", fwd, *call(q=q, q_out=q, **{name: T(5, 2, 64, ptr=5 * PLACE + 128)}))
    raises(f"'q_out' and 'q' {MATCH}", fwd, *call(q=q, q_out=T(5, 4, 64, ptr=5 * PLACE + 128)))
