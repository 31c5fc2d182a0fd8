"""The decode step's operators as they are used together: a decoder block that takes one
token at a time over a paged cache against the same block over the whole sequence; on side
streams, two calls at once, captured and replayed with eager work between, and two captured
graphs in turn."""

from __future__ import annotations

import dataclasses

import pytest
import torch

from custom_cuda_kernals_amd import kernels as K
from custom_cuda_kernals_amd._lib import native
from custom_cuda_kernals_amd.llama_block import CONFIGS, LlamaBlock, LlamaBlockConfig, PagedCache

pytestmark = pytest.mark.gpu

SMALL = LlamaBlockConfig(hidden_size=512, intermediate_size=1408, num_heads=8, num_kv_heads=2)  # heads of 64


def _block(mode, cfg=SMALL, seq=64):
    torch.manual_seed(0)
    ref = LlamaBlock(seq, cfg, mode="fused").eval()
    blk = LlamaBlock(seq, cfg, mode=mode).eval()
    blk.load_state_dict(ref.state_dict())
    return blk


def _tokens(b, s, hidden, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(b, s, hidden, dtype=torch.bfloat16, device="cuda", generator=g) * 0.5


def _off(got, want, x):
    """Relative difference of what the block adds to its input."""
    a, b = got.float() - x.float(), want.float() - x.float()
    return ((a - b).norm() / b.norm()).item()


@pytest.mark.parametrize("page_size", [16, 5])
@pytest.mark.parametrize("mode,limit", [("fused", 0.02), ("fp8", 0.08), ("fp8_block", 0.08)])
def test_decode_is_the_whole_sequence_a_token_at_a_time(mode, limit, page_size):
    """bf16 values between the kernels are rounded at other places, 2^-9 each: a hundredth of the update. Where FP8
    activations are quantised behind them, a rounding may take a code to its neighbour, 2^-4 of it."""
    blk, prompt, steps = _block(mode), 40, 20
    x = _tokens(3, prompt + steps, SMALL.hidden_size)
    with torch.no_grad():
        cache = PagedCache.allocate(SMALL, 3, 64, page_size)
        first = blk.prefill(x[:, :prompt].contiguous(), cache, *cache.advance(prompt))
        blk.rope_cos, blk.rope_sin = blk.rope_cos[:prompt].contiguous(), blk.rope_sin[:prompt].contiguous()
        assert _off(first, blk(x[:, :prompt].contiguous()), x[:, :prompt]) < limit
        whole = _block(mode, seq=prompt + steps)(x)
        for t in range(prompt, prompt + steps):
            y = blk.decode(x[:, t:t + 1].contiguous(), cache, *cache.advance(1))
            assert _off(y, whole[:, t:t + 1], x[:, t:t + 1]) < limit, t
    assert cache.lengths.tolist() == [60, 60, 60]


def test_decode_over_an_fp8_cache():
    blk = _block("fused")
    x = _tokens(2, 60, SMALL.hidden_size, 1)
    outs = []
    with torch.no_grad():
        for dtype, scale in ((torch.bfloat16, 1.0), (torch.float8_e4m3fn, 0.05)):
            cache = PagedCache.allocate(SMALL, 2, 64, dtype=dtype, key_scale=scale, value_scale=scale)
            blk.prefill(x[:, :59].contiguous(), cache, *cache.advance(59))
            outs.append(blk.decode(x[:, 59:].contiguous(), cache, *cache.advance(1)))
    # e4m3 rounds keys and values by 2^-4 at most; the block adds more than the attention
    assert 0 < _off(outs[1], outs[0], x[:, 59:]) < 0.1


def test_llama_3_8b_block():
    """The block at its own size, 4 sequences, one token after a prompt of 300."""
    cfg = CONFIGS["llama3-8b"]
    x = _tokens(4, 301, cfg.hidden_size, 2)
    with torch.no_grad():
        for mode, limit in (("fused", 0.02), ("fp8_block", 0.08)):
            blk = _block(mode, cfg, 301)
            cache = PagedCache.allocate(cfg, 4, 320)
            blk.prefill(x[:, :300].contiguous(), cache, *cache.advance(300))
            y = blk.decode(x[:, 300:].contiguous(), cache, *cache.advance(1))
            assert _off(y, blk(x)[:, 300:], x[:, 300:]) < limit, mode
            del blk
            torch.cuda.empty_cache()


def test_a_full_cache_keeps_what_it_has():
    """Tokens past a sequence's pages are not written anywhere."""
    blk, cfg = _block("fused"), SMALL
    cache = PagedCache.allocate(cfg, 2, 16)
    with torch.no_grad():
        x = _tokens(2, 16, cfg.hidden_size, 3)
        blk.prefill(x, cache, *cache.advance(16))
        keys = cache.keys.clone()
        positions, slots = cache.advance(1)
        assert positions.tolist() == [[16], [16]] and slots.tolist() == [[-1], [-1]]
        y = blk.decode(x[:, :1].contiguous(), cache, positions, slots)
    assert torch.equal(cache.keys, keys) and y.isfinite().all()


def test_refusals():
    blk, cache = _block("fused"), PagedCache.allocate(SMALL, 2, 16)
    x = _tokens(2, 2, SMALL.hidden_size)
    with pytest.raises(ValueError, match="one token a sequence"):
        blk.decode(x, cache, *cache.advance(2))
    with pytest.raises(ValueError, match="the cache's 2 sequences"):
        blk.decode(x[:1, :1], cache, *cache.advance(1))
    eager = LlamaBlock(8, SMALL, mode="eager")
    with pytest.raises(ValueError, match="has no cache"):
        eager.decode(x[:, :1], cache, *cache.advance(1))


def _replay(run, state, reset, times=4):
    """`run` captured and replayed, with eager runs and other work between; each replay against the eager result."""
    reset()
    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(times):
        for t in out:
            t.fill_(0)
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        reset()
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
        torch.empty(1 << 22, device="cuda").normal_()


@pytest.mark.parametrize("mode", ["fused", "fp8_block"])
def test_a_decode_step_replays_from_a_graph(mode):
    blk = _block(mode)
    x = _tokens(2, 30, SMALL.hidden_size, 4)
    cache = PagedCache.allocate(SMALL, 2, 64)
    with torch.no_grad():
        blk.prefill(x[:, :29].contiguous(), cache, *cache.advance(29))
        token = x[:, 29:].contiguous()

        def step():
            return [blk.decode(token, cache, *cache.advance(1))]

        _replay(step, cache, lambda: cache.lengths.fill_(29))


def _attention_case(seed, dtype=torch.bfloat16, b=3, context=900):
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-context // 16)
    q = torch.randn(b, 8, 64, device="cuda", generator=g).to(dtype)
    keys, values = (torch.randn(b * per, 16, 2, 64, device="cuda", generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(b * per, device="cuda", generator=g).view(b, per)
    lengths = torch.tensor([context, 17, context // 2][:b], device="cuda")
    return q, keys, values, table, lengths


def test_two_captured_graphs_in_turn():
    """Workspaces come from the caller's allocator: graphs that replay one after the other, and lengths that change
    between replays, as they do from token to token."""
    a, b = _attention_case(1), _attention_case(2)
    graphs, outs = [], []
    K.paged_attention(*a), K.paged_attention(*b)
    torch.cuda.synchronize()
    for case in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(K.paged_attention(*case, return_lse=True))
        graphs.append(graph)
    for n in (900, 33, 0, 512):
        for case in (a, b):
            case[4].fill_(n)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for case, out in zip((a, b), outs):
            want = K.paged_attention(*case, return_lse=True)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_two_calls_at_once():
    cases = [_attention_case(3 + i, context=3000) for i in range(2)]
    w = torch.randn(700, 512, device="cuda", dtype=torch.bfloat16)
    wc, ws = K.fp8_quant(w, "e4m3", "block")
    xs = [torch.randn(300, 512, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    frequencies, _ = K.rope_frequencies(64)
    heads = [torch.randn(500, 8, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
    positions = torch.arange(500, device="cuda")

    def work(i):
        return (K.paged_attention(*cases[i]), K.fp8_block_linear(*K.fp8_quant(xs[i], "e4m3", "group"), wc, ws),
                *K.rope_at(heads[i], heads[i][:, :2], positions, frequencies))

    want = [[t.clone() for t in work(i)] for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append(work(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w_ in zip(got, want) for a, b in zip(g, w_))


def test_launches_go_to_the_current_stream():
    q, keys, values, table, lengths = _attention_case(9)
    x = torch.randn(40, 512, device="cuda", dtype=torch.bfloat16)
    codes, scale = K.fp8_quant(x, "e4m3", "block")
    frequencies, _ = K.rope_frequencies(64)
    slots = torch.arange(3, device="cuda")
    k = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    calls = [lambda: K.paged_attention(q, keys, values, table, lengths), lambda: K.fp8_quant(x, "e4m3", "group"),
             lambda: K.fp8_block_linear(codes, scale, codes, scale), lambda: K.rope_at(q, k, slots, frequencies),
             lambda: K.rope_to_cache(q, k, k, keys, values, slots, slots, frequencies)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for call in calls:
        with torch.cuda.stream(side):
            call()
        assert native._last_launch_stream() == side.cuda_stream
        call()
        assert native._last_launch_stream() == torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()


def test_the_long_way_gives_the_same():
    """Calls that the one-call form leaves to the validating functions: under a default-device mode."""
    q, keys, values, table, lengths = _attention_case(10)
    x = torch.randn(40, 512, device="cuda", dtype=torch.bfloat16)
    codes, scale = K.fp8_quant(x, "e4m3", "group")
    wc, ws = K.fp8_quant(x, "e5m2", "block")
    frequencies, _ = K.rope_frequencies(64)
    positions = torch.arange(3, device="cuda")

    def calls():
        k2, v2 = keys.clone(), values.clone()
        turned = K.rope_to_cache(q, q[:, :2].contiguous(), q[:, 2:4].contiguous(), k2, v2, positions, positions, frequencies)
        return [K.paged_attention(q, keys, values, table, lengths),
                *K.paged_attention(q, keys, values, table, lengths, return_lse=True, window=100),
                *K.rope_at(q, q[:, :2].contiguous(), positions, frequencies), turned, k2, v2,
                K.fp8_block_linear(codes, scale, wc, ws), K.fp8_quant(x, "e4m3", "group")[1]]

    want = calls()
    with torch.device("cuda"):
        got = calls()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_named_and_requires_grad_inputs_record_nothing():
    x = torch.randn(5, 4, 64, device="cuda", requires_grad=True)
    frequencies, _ = K.rope_frequencies(64)
    out, _ = K.rope_at(x, x.detach().clone(), torch.arange(5, device="cuda"), frequencies)
    assert not out.requires_grad


def test_config_of_another_head_dim():
    cfg = dataclasses.replace(SMALL, num_heads=4, num_kv_heads=4)  # heads of 128
    blk = _block("fused", cfg, 33)
    x = _tokens(1, 33, cfg.hidden_size, 6)
    cache = PagedCache.allocate(cfg, 1, 40, page_size=7)
    with torch.no_grad():
        blk.prefill(x[:, :32].contiguous(), cache, *cache.advance(32))
        y = blk.decode(x[:, 32:].contiguous(), cache, *cache.advance(1))
        assert _off(y, blk(x)[:, 32:], x[:, 32:]) < 0.02


@pytest.mark.parametrize("op_id", ["rope_at", "paged_attention", "fp8_linear"])
def test_cli_targets(op_id):
    """The developer CLI's calls agree with their eager formulas: bf16 values, rounded once or twice each."""
    from custom_cuda_kernals_amd.cli.registry import REGISTRY

    target = REGISTRY[op_id].build_target("cuda")
    got, want = target.kernel(), target.eager()
    for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
        assert a.shape == b.shape and (a.float() - b.float()).norm() < 0.01 * b.float().norm()
