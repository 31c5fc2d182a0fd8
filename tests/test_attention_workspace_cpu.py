"""The scratch that an attention call asks for: none where a wave or a workgroup's waves
take each sequence, which is decided by the same rule as the launch, without a window. The
launcher refuses a missing workspace exactly where one is asked for, before any launch, so
that the calls here are only those it refuses."""

from __future__ import annotations

import ctypes

import pytest

from tests import _cck

F32, F16, BF16, E4M3 = 0, 1, 2, 3


@pytest.fixture(scope="module")
def lib():
    lib = _cck.load()
    lib.cck_paged_attention_workspace.restype = ctypes.c_int64
    lib.cck_paged_attention_workspace.argtypes = [ctypes.c_int64] * 6 + [ctypes.c_int32]
    return lib


@pytest.mark.parametrize("sequences,heads,kv,dim,page,width,cache", [
    (1024, 64, 64, 128, 16, 32, BF16),  # a wave each
    (1024, 64, 8, 128, 16, 32, BF16), (2048, 32, 8, 128, 16, 64, E4M3),  # a workgroup's waves
    (1, 32, 8, 128, 16, 2, BF16), (8, 32, 8, 128, 16, 16, F32), (64, 12, 12, 80, 13, 40, F16)])
def test_none_where_nothing_is_cut(lib, sequences, heads, kv, dim, page, width, cache):
    assert lib.cck_paged_attention_workspace(sequences, heads, kv, dim, page, width, cache) == 0


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("sequences,heads,kv,dim,page,width", [
    (1, 32, 8, 128, 16, 8192), (8, 32, 8, 128, 16, 512), (64, 32, 8, 128, 16, 512), (2, 64, 8, 256, 64, 300),
    (300, 12, 4, 80, 16, 1000), (2048, 8, 8, 16, 1, 9000)])
def test_some_where_sequences_are_cut(lib, sequences, heads, kv, dim, page, width, dtype):
    p = 1 << 20
    bytes_ = lib.cck_paged_attention_workspace(sequences, heads, kv, dim, page, width, dtype)
    # two parts a sequence at least, each a head's sums, their maximum and total; and two words a sequence
    assert bytes_ >= 2 * sequences * heads * (dim + 2) * 4 + 8 * sequences
    for workspace in (None, p + 4):
        assert lib.launch_paged_attention_fwd(p, p, p, p, p, p, None, workspace, heads * dim, dim, sequences, heads, kv, dim, 9,
                                              page, width, 0, 1.0, 1.0, 1.0, dtype, dtype, None) == 1


def test_wider_tables_never_ask_for_less(lib):
    """As the positions grow a wave, waves and then parts take a sequence, and never the other way round."""
    for sequences in (1, 7, 64, 500):
        for cache in (BF16, E4M3):
            asked = [lib.cck_paged_attention_workspace(sequences, 32, 8, 128, 16, w, cache) > 0 for w in range(1, 3000, 7)]
            assert asked == sorted(asked) and asked[-1] and not asked[0]
