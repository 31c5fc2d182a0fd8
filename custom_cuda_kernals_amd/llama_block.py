"""Llama-3-8B decoder block on the MI355X activation kernels - the path's
integration caller.

Same architecture and numbers as the reference's integration proof
(examples/llama_block.py:55-204): pre-norm, GQA 32/8 heads of 128, RoPE theta
500000, SwiGLU FFN 4096 -> 14336 -> 4096, rms eps 1e-5, bf16. Four variants
share one set of weights:

* ``"eager"`` - plain torch ops (the reference's BaselineLlamaBlock);
* ``"fused"`` - the reference's CustomCUDA_LlamaBlock with this library:
  fused RMSNorm + residual, in-place RoPE and SwiGLU; GEMMs in bf16;
* ``"fp8"``   - the MI355X FP8 path: RMSNorm + residual fused with per-token
  FP8 quantisation feeds FP8 q/k/v and gate/up GEMMs (torch._scaled_mm on
  hipBLASLt, OCP e4m3fn, row-wise activation scales x per-output-channel
  weight scales); SwiGLU fused with per-token FP8 feeds the FP8 down
  projection; the attention output is quantised per token for the FP8 o_proj.
  Weights are quantised once, per output channel, with this library's
  per-token quantiser (a weight row is an output channel);
* ``"fp8_block"`` - FP8 with a scale for each block of 128 (``fp8_block_linear``):
  weights in 128 x 128 tiles, activations one scale for 128 neighbours of a token,
  behind the bf16 RMSNorm and SwiGLU.

Attention over a whole sequence (scaled_dot_product_attention) is identical in all.

Serving (not ``"eager"``): ``prefill`` writes a prompt's keys and values into a
``PagedCache``, ``decode`` takes one new token a sequence through the block over it
(``rope_to_cache``, ``paged_attention``)::

    cache = PagedCache.allocate(block.cfg, sequences=8, max_length=4096)
    y = block.prefill(prompt, cache, *cache.advance(prompt.shape[1]))
    y = block.decode(token, cache, *cache.advance(1))  # token [8, 1, hidden]
"""

from __future__ import annotations

import dataclasses
import statistics

import torch
import torch.nn as nn
import torch.nn.functional as F

from custom_cuda_kernals_amd.fp8_format import fp8_linear
from custom_cuda_kernals_amd.kernels import (
    fp8_block_linear,
    fp8_quant,
    paged_attention,
    rmsnorm_residual,
    rmsnorm_residual_fp8,
    rope,
    rope_at,
    rope_frequencies,
    rope_to_cache,
    swiglu,
    swiglu_fp8,
)

__all__ = ["LlamaBlockConfig", "LlamaBlock", "PagedCache", "rope_tables", "block_latency_ms", "MODES", "CONFIGS"]

MODES = ("eager", "fused", "fp8", "fp8_block")


@dataclasses.dataclass(frozen=True)
class LlamaBlockConfig:
    """Llama-3-8B config.json values (reference examples/llama_block.py:55-71)."""

    hidden_size: int = 4096
    intermediate_size: int = 14336
    num_heads: int = 32
    num_kv_heads: int = 8
    rms_eps: float = 1e-5
    rope_theta: float = 500000.0

    @property
    def head_dim(self) -> int:
        return self.hidden_size // self.num_heads


# The reference's block (Llama-3-8B) and, as an addition, Llama-3-70B's layer
# shapes (config.json: hidden 8192, intermediate 28672, 64 heads, 8 KV heads).
CONFIGS = {
    "llama3-8b": LlamaBlockConfig(),
    "llama3-70b": LlamaBlockConfig(hidden_size=8192, intermediate_size=28672, num_heads=64, num_kv_heads=8),
}


@dataclasses.dataclass
class PagedCache:
    """Keys and values of one layer in pages, and where each sequence's are. Layers share
    ``page_table`` and ``lengths``; one ``advance`` a step serves them all."""

    keys: torch.Tensor  # [pages, page_size, kv_heads, head_dim]; of the block's dtype, or FP8
    values: torch.Tensor
    page_table: torch.Tensor  # int64 [sequences, pages of each]; -1: none
    lengths: torch.Tensor  # int64 [sequences]
    key_scale: float = 1.0  # of FP8 keys and values
    value_scale: float = 1.0

    @classmethod
    def allocate(cls, cfg: LlamaBlockConfig, sequences: int, max_length: int, page_size: int = 16,
                 dtype: torch.dtype = torch.bfloat16, device: str = "cuda", key_scale: float = 1.0,
                 value_scale: float = 1.0) -> "PagedCache":
        """An empty cache in which each sequence has all its pages."""
        each = -(-max_length // page_size)
        shape = (sequences * each, page_size, cfg.num_kv_heads, cfg.head_dim)
        keys, values = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
        table = torch.arange(sequences * each, device=device).view(sequences, each)
        return cls(keys, values, table, torch.zeros(sequences, dtype=torch.int64, device=device), key_scale, value_scale)

    def advance(self, tokens: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Makes every sequence ``tokens`` longer: the new tokens' positions and slots, int64
        ``[sequences, tokens]``. Past a sequence's pages the slot is -1: such a token's keys and values
        are not kept. Nothing waits for the GPU, and ``lengths`` changes in place."""
        page_size, each = self.keys.shape[1], self.page_table.shape[1]
        positions = self.lengths[:, None] + torch.arange(tokens, device=self.lengths.device)
        index = positions // page_size
        pages = self.page_table.gather(1, index.clamp(max=each - 1))
        slots = torch.where((index < each) & (pages >= 0), pages * page_size + positions % page_size, -1)
        self.lengths += tokens
        return positions, slots


def rope_tables(seq_len: int, head_dim: int, theta: float, device) -> tuple[torch.Tensor, torch.Tensor]:
    """fp32 [S, D/2] cos/sin tables, computed as the reference's
    compute_cos_sin (baselines/rope.py:103-115)."""
    exponents = torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim
    inv_freq = 1.0 / (theta ** exponents)
    angles = torch.outer(torch.arange(seq_len, dtype=torch.float32, device=device), inv_freq)
    return angles.cos().contiguous(), angles.sin().contiguous()


def _eager_rmsnorm_residual(x, residual, weight, eps):
    ro = x + residual
    r32 = ro.float()
    normed = r32 * torch.rsqrt(r32.pow(2).mean(-1, keepdim=True) + eps)
    return normed.to(x.dtype) * weight, ro


def _eager_rope(q, k, cos, sin):
    def rot(t):
        t32 = t.float()
        half = t32.shape[-1] // 2
        a, b = t32[..., :half], t32[..., half:]
        c, s = cos[None, :, None, :], sin[None, :, None, :]
        return torch.cat([a * c - b * s, b * c + a * s], dim=-1).to(t.dtype)

    return rot(q), rot(k)


def _eager_swiglu(gate, up):
    g32 = gate.float()
    return (g32 * torch.sigmoid(g32)).to(gate.dtype) * up


class _Fp8Linear:
    """A bf16 weight [N, K] quantised once to e4m3fn per output channel; the
    activation comes per token (row-wise x row-wise _scaled_mm)."""

    def __init__(self, weight: torch.Tensor) -> None:
        self.w_codes, self.w_scale = fp8_quant(weight.contiguous(), "e4m3", "token")

    def __call__(self, x_fp8: torch.Tensor, x_scale: torch.Tensor) -> torch.Tensor:
        return fp8_linear(x_fp8, x_scale, "token", self.w_codes, self.w_scale, "token")


class _BlockFp8Linear:
    """A bf16 weight [N, K] quantised once to e4m3fn in 128 x 128 tiles; the activation in
    groups of 128 neighbours of a token."""

    def __init__(self, weight: torch.Tensor) -> None:
        self.w_codes, self.w_scale = fp8_quant(weight.contiguous(), "e4m3", "block")

    def __call__(self, x_fp8: torch.Tensor, x_scale: torch.Tensor) -> torch.Tensor:
        return fp8_block_linear(x_fp8, x_scale, self.w_codes, self.w_scale)


class LlamaBlock(nn.Module):
    def __init__(self, seq_len: int, cfg: LlamaBlockConfig = LlamaBlockConfig(), mode: str = "fused",
                 dtype: torch.dtype = torch.bfloat16, device: str = "cuda") -> None:
        super().__init__()
        if mode not in MODES:
            raise ValueError(f"mode must be one of {MODES}, got {mode!r}")
        self.cfg, self.mode = cfg, mode
        h, i, d = cfg.hidden_size, cfg.intermediate_size, cfg.head_dim

        def linear(n_in, n_out):
            return nn.Linear(n_in, n_out, bias=False, dtype=dtype, device=device)

        self.input_layernorm_weight = nn.Parameter(torch.ones(h, dtype=dtype, device=device))
        self.post_attention_layernorm_weight = nn.Parameter(torch.ones(h, dtype=dtype, device=device))
        self.q_proj, self.k_proj = linear(h, cfg.num_heads * d), linear(h, cfg.num_kv_heads * d)
        self.v_proj, self.o_proj = linear(h, cfg.num_kv_heads * d), linear(cfg.num_heads * d, h)
        self.gate_proj, self.up_proj, self.down_proj = linear(h, i), linear(h, i), linear(i, h)
        cos, sin = rope_tables(seq_len, d, cfg.rope_theta, device)
        self.register_buffer("rope_cos", cos, persistent=False)
        self.register_buffer("rope_sin", sin, persistent=False)
        self.register_buffer("rope_frequencies", rope_frequencies(d, cfg.rope_theta, device=device)[0], persistent=False)
        self._fp8 = None

    def prepare_fp8(self) -> None:
        """Quantise the projection weights (call after loading weights)."""
        linear = _BlockFp8Linear if self.mode == "fp8_block" else _Fp8Linear
        self._fp8 = {name: linear(getattr(self, name).weight.detach())
                     for name in ("q_proj", "k_proj", "v_proj", "o_proj", "gate_proj", "up_proj", "down_proj")}

    def _attention(self, q, k, v):
        b, s = q.shape[0], q.shape[1]
        rep = self.cfg.num_heads // self.cfg.num_kv_heads
        k = k.repeat_interleave(rep, dim=2)
        v = v.repeat_interleave(rep, dim=2)
        out = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
        return out.transpose(1, 2).reshape(b, s, -1)

    def _project(self, x: torch.Tensor) -> tuple[torch.Tensor, ...]:
        """q, k and v of the normalised x, and the residual."""
        cfg = self.cfg
        b, s, hid = x.shape
        zero = torch.zeros_like(x)
        if self.mode == "fp8":
            hq, hs, residual = rmsnorm_residual_fp8(x, zero, self.input_layernorm_weight, cfg.rms_eps)
            linear = self._linears(hq.view(b * s, hid), hs.view(b * s))
        else:
            norm = _eager_rmsnorm_residual if self.mode == "eager" else rmsnorm_residual
            h, residual = norm(x, zero, self.input_layernorm_weight, cfg.rms_eps)
            linear = self._linears(h)
        q = linear("q_proj").view(b, s, cfg.num_heads, cfg.head_dim)
        k = linear("k_proj").view(b, s, cfg.num_kv_heads, cfg.head_dim)
        v = linear("v_proj").view(b, s, cfg.num_kv_heads, cfg.head_dim)
        return q, k, v, residual

    def _linears(self, h: torch.Tensor, scale: torch.Tensor | None = None):
        """The projections of h by name; of FP8 codes with their scale, or of bf16 values."""
        if self.mode in ("eager", "fused"):
            return lambda name: getattr(self, name)(h)
        if self._fp8 is None:
            self.prepare_fp8()
        if scale is None:
            h, scale = fp8_quant(h.reshape(-1, h.shape[-1]), "e4m3", "group" if self.mode == "fp8_block" else "token")
        return lambda name: self._fp8[name](h, scale)

    def _finish(self, a: torch.Tensor, residual: torch.Tensor) -> torch.Tensor:
        """From the attention's output [b, s, heads * head_dim] to the block's."""
        cfg = self.cfg
        b, s, hid = residual.shape
        attn = self._linears(a)("o_proj").view(b, s, hid)
        if self.mode == "fp8":
            h2q, h2s, residual2 = rmsnorm_residual_fp8(attn, residual, self.post_attention_layernorm_weight, cfg.rms_eps)
            linear = self._linears(h2q.view(b * s, hid), h2s.view(b * s))
            mq, ms = swiglu_fp8(linear("gate_proj"), linear("up_proj"), "e4m3")
            return self._linears(mq, ms)("down_proj").view(b, s, hid) + residual2
        norm = _eager_rmsnorm_residual if self.mode == "eager" else rmsnorm_residual
        h2, residual2 = norm(attn, residual, self.post_attention_layernorm_weight, cfg.rms_eps)
        linear = self._linears(h2)
        gate, up = linear("gate_proj"), linear("up_proj")
        act = _eager_swiglu(gate, up) if self.mode == "eager" else swiglu(gate, up)
        return self._linears(act)("down_proj").view(b, s, hid) + residual2

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        q, k, v, residual = self._project(x)
        if self.mode == "eager":
            q, k = _eager_rope(q, k, self.rope_cos, self.rope_sin)
        else:
            q, k = rope(q, k, self.rope_cos, self.rope_sin, inplace=True)
        return self._finish(self._attention(q, k, v), residual)

    def _check_serving(self, x: torch.Tensor, cache: PagedCache) -> None:
        if self.mode == "eager":
            raise ValueError("the eager block has no cache: use mode 'fused', 'fp8' or 'fp8_block'")
        if x.dim() != 3 or x.shape[0] != cache.lengths.shape[0]:
            raise ValueError(f"x must be [sequences, tokens, hidden] with the cache's {cache.lengths.shape[0]} sequences, "
                             f"got {tuple(x.shape)}")

    def prefill(self, x: torch.Tensor, cache: PagedCache, positions: torch.Tensor, slots: torch.Tensor,
                check: bool = True) -> torch.Tensor:
        """``forward`` of prompts ``[sequences, tokens, hidden]`` from position 0 on (of an empty cache), their keys
        and values kept in ``cache``; positions and slots from its ``advance``, which makes all prompts equally long.
        The prompt alone is attended to, so positions further on are refused. To tell, a call waits for the GPU, but not
        while a graph is captured, nor with ``check=False``: of many layers the first one's check is enough."""
        self._check_serving(x, cache)
        if check and not torch.cuda.is_current_stream_capturing() and bool(positions[..., :1].any()):
            raise ValueError("prefill takes prompts from position 0 on, over an empty cache: what the cache holds would not "
                             "be attended to")
        q, k, v, residual = self._project(x)
        rope_to_cache(q, k, v, cache.keys, cache.values, slots, positions, self.rope_frequencies,
                      key_scale=cache.key_scale, value_scale=cache.value_scale, inplace=True)
        # The cache's keys are turned; those of this call's own attention are turned here.
        k, _ = rope_at(k, k[:, :, :0], positions, self.rope_frequencies)
        return self._finish(self._attention(q, k, v), residual)

    def decode(self, x: torch.Tensor, cache: PagedCache, positions: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
        """One new token of each sequence, x ``[sequences, 1, hidden]``, at its position over all that ``cache``
        holds; positions and slots from its ``advance(1)``."""
        self._check_serving(x, cache)
        if x.shape[1] != 1:
            raise ValueError(f"decode takes one token a sequence, got {x.shape[1]}")
        q, k, v, residual = self._project(x)
        q = rope_to_cache(q, k, v, cache.keys, cache.values, slots, positions, self.rope_frequencies,
                          key_scale=cache.key_scale, value_scale=cache.value_scale, inplace=True)
        a = paged_attention(q.squeeze(1), cache.keys, cache.values, cache.page_table, cache.lengths,
                            key_scale=cache.key_scale, value_scale=cache.value_scale)
        return self._finish(a.view(x.shape[0], 1, -1), residual)


def block_latency_ms(block: nn.Module, x: torch.Tensor, warmup: int = 5, iters: int = 20,
                     flush_bytes: int = 1 << 30) -> dict:
    """Median / IQR of block(x) in ms, with the reference's methodology
    (examples/llama_block.py:220-250): a cache flush before every measured
    iteration (1 GiB here, larger than MI355X's 256 MB Infinity Cache) and
    HIP events around the forward."""
    flush = torch.empty(flush_bytes // 4, dtype=torch.float32, device=x.device)
    times = []
    with torch.no_grad():
        for _ in range(warmup):
            block(x)
        torch.cuda.synchronize()
        for _ in range(iters):
            flush.fill_(1.0)
            torch.cuda.synchronize()
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            block(x)
            end.record()
            torch.cuda.synchronize()
            times.append(start.elapsed_time(end))
        torch.cuda.reset_peak_memory_stats()
        block(x)
        torch.cuda.synchronize()
        peak = torch.cuda.max_memory_allocated()
    times.sort()
    return {"median_ms": round(statistics.median(times), 4),
            "iqr_ms": round(times[(3 * len(times)) // 4] - times[len(times) // 4], 4),
            "peak_mem_MB": round(peak / 2**20, 1)}
