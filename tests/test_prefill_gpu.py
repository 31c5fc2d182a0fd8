"""Where a prompt may go: LlamaBlock.prefill attends to the prompt alone, so it takes no
prompt behind positions that a cache holds."""

from __future__ import annotations

import pytest
import torch

from custom_cuda_kernals_amd.llama_block import PagedCache
from tests.test_decode_use_gpu import SMALL, _block, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["fused", "fp8", "fp8_block"])
def test_a_second_prompt_is_refused(mode):
    blk, x = _block(mode), _tokens(2, 20, SMALL.hidden_size)
    with torch.no_grad():
        cache = PagedCache.allocate(SMALL, 2, 64)
        first = blk.prefill(x, cache, *cache.advance(20))
        kept = cache.keys.clone(), cache.values.clone()
        with pytest.raises(ValueError, match="from position 0 on"):
            blk.prefill(x, cache, *cache.advance(20))
        assert torch.equal(cache.keys, kept[0]) and torch.equal(cache.values, kept[1])
        cache.lengths.zero_()  # emptied
        at = cache.advance(20)
        assert torch.equal(blk.prefill(x, cache, *at), first) and torch.equal(blk.prefill(x, cache, *at, check=False), first)


def test_one_sequence_of_many():
    """Refused if a single sequence holds something."""
    blk, x = _block("fused"), _tokens(3, 4, SMALL.hidden_size)
    cache = PagedCache.allocate(SMALL, 3, 64)
    cache.lengths[1] = 1
    with torch.no_grad(), pytest.raises(ValueError, match="from position 0 on"):
        blk.prefill(x, cache, *cache.advance(4))


def test_a_prompt_into_a_graph():
    blk, x = _block("fused"), _tokens(2, 20, SMALL.hidden_size)
    cache = PagedCache.allocate(SMALL, 2, 64)
    with torch.no_grad():
        want = blk.prefill(x, cache, *cache.advance(20))
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.lengths.zero_()
            got = blk.prefill(x, cache, *cache.advance(20))
        for _ in range(3):
            got.fill_(0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want) and cache.lengths.tolist() == [20, 20]
