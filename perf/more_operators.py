"""Workloads of the decode step, for timing them and comparing their outputs.

``listed()`` names the calls that serving a decoder block (and training its
rotary positions) makes of ``custom_cuda_kernals_amd.kernels``: rotation at
given positions and its gradient, rotation with the write of keys and values
into a paged cache, attention of one new token a sequence over that cache, and
the FP8 product with a scale for each block of 128. ``draw(rng)`` gives another
case of the same ranges. ``prepare`` makes a case's inputs on the GPU from a
seed, ``run`` is one pass (``own``: the package's kernels, else elementary torch
operations in float32), ``exact`` is the result in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn,
          "e5m2": torch.float8_e5m2}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1, "e5m2": 1}
FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
TILE = 128
CACHE_SCALE = 0.25  # of keys and values in an FP8 cache


def listed() -> list[dict]:
    return [
        # A decode step of 16 sequences at the Llama-3-8B block's heads, at positions up to 128 Ki.
        {"name": "rope_decode", "op": "rope", "tokens": 16, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "layout": "half", "scaling": "parts", "context": 131072, "inverse": False, "dtype": "bf16"},
        # The gradient of a training step of 8 x 4096 packed tokens.
        {"name": "rope_grad", "op": "rope", "tokens": 32768, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "layout": "half", "scaling": "none", "context": 4096, "inverse": True, "dtype": "bf16"},
        # Interleaved pairs on part of a head, an odd number of tokens, float32.
        {"name": "rope_partial", "op": "rope", "tokens": 1003, "heads": 12, "kv_heads": 12, "dim": 80, "rotary": 52,
         "layout": "interleaved", "scaling": "yarn", "context": 32768, "inverse": False, "dtype": "fp32"},
        # The same decode step, its keys and values going to an FP8 cache.
        {"name": "cache_decode", "op": "cache", "tokens": 64, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "layout": "half", "scaling": "parts", "context": 131072, "page": 16, "cache": "e4m3", "dtype": "bf16"},
        # A prompt of 8192 tokens to a cache of its own type.
        {"name": "cache_prompt", "op": "cache", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rotary": 128,
         "layout": "half", "scaling": "none", "context": 8192, "page": 16, "cache": "bf16", "dtype": "bf16"},
        # Attention of one sequence's next token, 700 tokens in: latency.
        {"name": "attention_one", "op": "attention", "sequences": 1, "context": 700, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "cache": "bf16", "dtype": "bf16"},
        # A batch of 64 sequences of up to 8192 tokens (one of them empty, a padded row).
        {"name": "attention_batch", "op": "attention", "sequences": 64, "context": 8192, "ragged": True, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "window": 0, "cache": "bf16", "dtype": "bf16"},
        # Two long contexts at Llama-3-70B's heads over an FP8 cache.
        {"name": "attention_long", "op": "attention", "sequences": 2, "context": 131072, "ragged": False, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "cache": "e4m3", "dtype": "bf16"},
        # Every head its own keys, an odd page, heads of 80, a window.
        {"name": "attention_odd", "op": "attention", "sequences": 7, "context": 3001, "ragged": True, "heads": 12,
         "kv_heads": 12, "dim": 80, "page": 13, "window": 1000, "cache": "fp16", "dtype": "fp16"},
        # A decode step of 8 sequences through the up projection of the Llama-3-8B FFN.
        {"name": "linear_decode", "op": "linear", "tokens": 8, "top_k": 1, "experts": 0, "n": 14336, "k": 4096,
         "x_scale": "group", "format": "e4m3", "dtype": "bf16"},
        # Prefill of 8192 tokens through it.
        {"name": "linear_prefill", "op": "linear", "tokens": 8192, "top_k": 1, "experts": 0, "n": 14336, "k": 4096,
         "x_scale": "group", "format": "e4m3", "dtype": "bf16"},
        # Gradients in e5m2, 128 x 128 tiles, of ragged experts with odd widths.
        {"name": "linear_experts", "op": "linear", "tokens": 777, "top_k": 2, "experts": 8, "n": 1412, "k": 1030,
         "x_scale": "block", "format": "e5m2", "dtype": "fp32"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng) -> dict:
    kv = rng.choice([1, 2, 4, 8, 8, 12, 32])
    return {"heads": kv * rng.choice([1, 1, 3, 4, 4, 7, 8, 16] if kv <= 8 else [1, 2]), "kv_heads": kv,
            "dim": rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])}


def _rotary(rng, dim: int) -> dict:
    return {"rotary": dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2),
            "layout": rng.choice(["half", "half", "interleaved"]),
            "scaling": rng.choice(["none", "linear", "ntk", "parts", "yarn"]), "context": _log_int(rng, 16, 1 << 20)}


def draw(rng) -> dict:
    op = rng.choice(["rope", "cache", "attention", "attention", "attention", "linear", "linear", "linear"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("rope", "cache"):
        case = {"op": op, "tokens": 0, **_heads(rng)}
        case |= _rotary(rng, case["dim"])
        row = (case["heads"] + case["kv_heads"]) * case["dim"] * SIZES[dtype]
        most = 32768 * 40 * 128 * 2 if op == "rope" else 8192 * 40 * 128 * 2
        case["tokens"] = _log_int(rng, 1, max(1, most // row))
        if op == "rope":
            return {**case, "inverse": rng.random() < 0.5, "dtype": dtype}
        return {**case, "page": rng.choice([1, 8, 13, 16, 16, 64, 128]), "cache": rng.choice([dtype, dtype, "e4m3", "e5m2"]),
                "dtype": dtype}
    if op == "attention":
        case = {"op": op, "sequences": _log_int(rng, 1, 256), "context": 0, "ragged": rng.random() < 0.6, **_heads(rng),
                "page": rng.choice([1, 8, 13, 16, 16, 32, 64, 256]), "window": 0,
                "cache": rng.choice([dtype, dtype, "e4m3", "e5m2"]), "dtype": dtype}
        row = case["kv_heads"] * case["dim"] * max(2, SIZES[dtype])
        most = 64 * 8192 * 8 * 128 * 2 // (2 if not case["ragged"] else 1) // (row * case["sequences"])
        case["context"] = _log_int(rng, 1, max(1, min(most, 1 << 18)))
        # No more scores than the largest listed case has.
        while case["sequences"] * case["context"] * case["heads"] > 64 * 8192 * 32:
            case["context"] //= 2
        if rng.random() < 0.25:
            case["window"] = rng.randint(1, case["context"])
        return case
    experts = rng.choice([0, 0, 8, 16, 64, rng.randint(1, 128)])
    top_k = rng.randint(1, min(6, experts)) if experts else 1
    width = [768, 1024, 1408, 1536, 2048, 2560, 4096, 5120, 7168, 8192, 14336]
    case = {"op": op, "tokens": _log_int(rng, 1, 8192 // top_k), "top_k": top_k, "experts": experts,
            "n": rng.choice(width) if rng.random() < 0.6 else _log_int(rng, 33, 12000),
            "k": rng.choice(width) if rng.random() < 0.6 else _log_int(rng, 33, 12000),
            "x_scale": rng.choice(["group", "group", "block"]), "format": rng.choice(["e4m3", "e4m3", "e5m2"]),
            "dtype": dtype}
    # No more weights, and no more products, than the largest listed case of each kind has.
    while max(experts, 1) * case["n"] * case["k"] > 8 * 14336 * 4096 or (
            case["tokens"] * top_k * case["n"] * case["k"] > 8192 * 14336 * 4096):
        case["n"], case["k"] = max(33, case["n"] * 2 // 3), max(33, case["k"] * 2 // 3)
    return case


def _lengths(case: dict) -> list[int]:
    """Of each sequence; ragged ones from nothing up to the whole context."""
    n, context = case["sequences"], case["context"]
    if not case["ragged"]:
        return [context] * n
    return [context] if n == 1 else [context * i // (n - 1) for i in range(n)]


def _active(case: dict) -> float:
    """Experts that some token is expected to reach."""
    e = case["experts"]
    return e * (1.0 - (1.0 - case["top_k"] / e) ** case["tokens"]) if e else 1.0


def work(case: dict) -> dict:
    size = SIZES[case["dtype"]]
    if case["op"] == "linear":
        rows, n, k = case["tokens"] * case["top_k"], case["n"], case["k"]
        # activations in, quantised, to y; the codes between are the path's own
        return {"bytes": rows * (k + n) * size + _active(case) * n * k, "flops": 2 * rows * n * k}
    q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    if case["op"] == "rope":
        return {"bytes": case["tokens"] * (2 * (q + kv) * size + 8),
                "flops": 3 * case["tokens"] * case["rotary"] * (case["heads"] + case["kv_heads"])}
    if case["op"] == "cache":
        return {"bytes": case["tokens"] * (2 * (q + kv) * size + 2 * kv * SIZES[case["cache"]] + 16),
                "flops": 3 * case["tokens"] * case["rotary"] * (case["heads"] + case["kv_heads"])}
    seen = sum(min(n, case["window"] or n) for n in _lengths(case))
    return {"bytes": 2 * seen * kv * SIZES[case["cache"]] + case["sequences"] * (2 * q * size + 4 * case["heads"]),
            "flops": 4 * seen * q}


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------

def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, std: float, dtype: torch.dtype, gen: torch.Generator) -> torch.Tensor:
    return (torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen) * std).to(dtype)


def _frequencies(case: dict) -> tuple[torch.Tensor, float]:
    """Angles a position, in float64, and the factor of the rotated elements. The
    formulas of scaling for long contexts: positions divided by a factor (linear), a
    larger base (ntk), or each frequency between itself and the divided one by how often
    it turns within the original length (parts, and yarn with its factor)."""
    dim, theta, factor, original = case["rotary"], 500000.0, 8.0, 8192
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    kind = case["scaling"]
    if kind == "ntk" and dim > 2:
        theta = theta * factor ** (dim / (dim - 2))
    f = theta ** (-i / dim)
    if kind == "linear":
        f = f / factor
    if kind in ("parts", "yarn"):
        low, high = (1.0, 4.0) if kind == "parts" else (1.0, 32.0)
        keep = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f / factor * (1 - keep) + f * keep
    return f.cuda(), 0.1 * math.log(factor) + 1.0 if kind == "yarn" else 1.0


def _scale(amax: torch.Tensor, fmt: str) -> torch.Tensor:
    """amax / FP8_MAX, divided: by a number torch multiplies with its reciprocal."""
    return (amax / torch.full_like(amax, FP8_MAX[fmt])).clamp(min=1e-12)


def _quant_tiles(w: torch.Tensor, fmt: str) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of 128 x 128 tiles of the last two dimensions."""
    n, k = w.shape[-2:]
    rows, cols = -(-n // TILE), -(-k // TILE)
    v = torch.nn.functional.pad(w.float(), (0, cols * TILE - k, 0, rows * TILE - n))
    v = v.unflatten(-1, (cols, TILE)).unflatten(-3, (rows, TILE))
    scale = _scale(v.abs().amax(dim=(-3, -1)), fmt)
    codes = (v / scale[..., :, None, :, None]).flatten(-4, -3).flatten(-2)[..., :n, :k]
    return codes.to(DTYPES[fmt]).contiguous(), scale.contiguous()


def _routing(case: dict, gen: torch.Generator) -> tuple[torch.Tensor, list[int]]:
    """Offsets of the experts' rows, as routing gives them: some experts are liked
    more than others, and few tokens leave some without any."""
    e, t = case["experts"], case["tokens"]
    logits = torch.randn((t, e), device="cuda", generator=gen) + 0.3 * torch.randn(e, device="cuda", generator=gen)
    sizes = torch.bincount(logits.topk(case["top_k"], dim=-1).indices.flatten(), minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = sizes.cumsum(0)
    return offsets, sizes.tolist()


def _prepare_linear(case: dict, gen: torch.Generator) -> dict:
    rows, n, k, e = case["tokens"] * case["top_k"], case["n"], case["k"], case["experts"]
    x = torch.randn((rows, k), device="cuda", generator=gen)
    far = torch.rand((rows, k), device="cuda", generator=gen) < 1e-3  # one value in a thousand 20 times as large
    state = {"op": "linear", "x": torch.where(far, x * 20.0, x).to(DTYPES[case["dtype"]]), "format": case["format"],
             "x_scale": case["x_scale"], "offsets": None, "sizes": [rows]}
    if e:
        state["offsets"], state["sizes"] = _routing(case, gen)
    w = [_quant_tiles(_normal((n, k), 0.02, torch.bfloat16, gen), "e4m3") for _ in range(max(e, 1))]
    state["w"], state["ws"] = (torch.stack(p) if e else p[0] for p in zip(*w))
    return state


def prepare(case: dict, seed: int) -> dict:
    gen = _gen(seed)
    if case["op"] == "linear":
        return _prepare_linear(case, gen)
    dtype, heads, kv, dim = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]
    state = {"op": case["op"], "dtype": dtype}
    if case["op"] in ("rope", "cache"):
        t = case["tokens"]
        state["frequencies"], state["factor"] = _frequencies(case)
        state |= {"layout": case["layout"], "inverse": case.get("inverse", False),
                  "positions": torch.randint(0, case["context"], (t,), device="cuda", generator=gen),
                  "q": _normal((t, heads, dim), 1.0, dtype, gen), "k": _normal((t, kv, dim), 1.0, dtype, gen)}
        if case["op"] == "cache":
            # The tokens' slots are anywhere in a cache of about twice as many.
            page, cached = case["page"], DTYPES[case["cache"]]
            pages = 2 * t // page + 2
            state |= {"v": _normal((t, kv, dim), 1.0, dtype, gen),
                      "slots": torch.randperm(pages * page, device="cuda", generator=gen)[:t],
                      "cache_scale": CACHE_SCALE if SIZES[case["cache"]] == 1 else 1.0,
                      "keys": torch.zeros((pages, page, kv, dim), device="cuda").to(cached),
                      "values": torch.zeros((pages, page, kv, dim), device="cuda").to(cached)}
        return state
    b, page, cached = case["sequences"], case["page"], DTYPES[case["cache"]]
    scale = CACHE_SCALE if SIZES[case["cache"]] == 1 else 1.0
    per = -(-case["context"] // page)
    pages = b * per + 3  # each sequence has pages of its own, anywhere in the cache
    lengths = torch.tensor(_lengths(case), device="cuda")[torch.randperm(b, device="cuda", generator=gen)]
    table = torch.randperm(pages, device="cuda", generator=gen)[:b * per].view(b, per)
    return {**state, "lengths": lengths, "table": table, "window": case["window"], "cache_scale": scale,
            "q": _normal((b, heads, dim), 1.5, dtype, gen),  # some positions stand out
            "keys": _normal((pages, page, kv, dim), 1.0 / scale, cached, gen),
            "values": _normal((pages, page, kv, dim), 1.0 / scale, cached, gen)}


# ---------------------------------------------------------------------------
# One pass: the package's kernels, or the plain form.
# ---------------------------------------------------------------------------

def _own(s: dict):
    from custom_cuda_kernals_amd import kernels as K

    if s["op"] == "rope":
        return K.rope_at(s["q"], s["k"], s["positions"], s["frequencies"], layout=s["layout"], scale=s["factor"],
                         inverse=s["inverse"])
    if s["op"] == "cache":
        q = K.rope_to_cache(s["q"], s["k"], s["v"], s["keys"], s["values"], s["slots"], s["positions"], s["frequencies"],
                            layout=s["layout"], scale=s["factor"], key_scale=s["cache_scale"],
                            value_scale=s["cache_scale"])
        return q, s["keys"], s["values"]
    if s["op"] == "attention":
        return K.paged_attention(s["q"], s["keys"], s["values"], s["table"], s["lengths"], window=s["window"],
                                 key_scale=s["cache_scale"], value_scale=s["cache_scale"], return_lse=True)
    codes, scale = K.fp8_quant(s["x"], s["format"], s["x_scale"])
    return K.fp8_block_linear(codes, scale, s["w"], s["ws"], s["offsets"], s["x"].dtype)


def _rotated(x: torch.Tensor, s: dict) -> torch.Tensor:
    """float32, the angles in float64."""
    angle = s["positions"].double()[:, None] * s["frequencies"]
    cos, sin = (angle.cos() * s["factor"]).float()[:, None], (angle.sin() * s["factor"]).float()[:, None]
    sin = -sin if s["inverse"] else sin
    x = x.float()
    rot = 2 * s["frequencies"].numel()
    if s["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], dim=-1)


def _cached(x: torch.Tensor, cache: torch.Tensor, scale: float) -> torch.Tensor:
    """float32 values in a cache's type: FP8 divided by the scale, no further than its largest."""
    if cache.element_size() == 1:
        top = torch.finfo(cache.dtype).max
        x = (x / scale).clamp(-top, top)
    return x.to(cache.dtype)


def _attention(s: dict):
    b, heads, dim = s["q"].shape
    per, page, kv = s["table"].shape[1], s["keys"].shape[1], s["keys"].shape[2]
    at = torch.arange(per * page, device="cuda")
    seen = at < s["lengths"][:, None]
    if s["window"]:
        seen = seen & (at >= s["lengths"][:, None] - s["window"])
    k = (s["keys"][s["table"]].float() * s["cache_scale"]).flatten(1, 2).transpose(1, 2)  # [b, kv, length, dim]
    v = (s["values"][s["table"]].float() * s["cache_scale"]).flatten(1, 2).transpose(1, 2)
    q = s["q"].float().view(b, kv, heads // kv, dim)
    scores = torch.matmul(q, k.transpose(2, 3)) * dim ** -0.5
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / total.clamp(min=1e-30)
    return out.view(b, heads, dim).to(s["dtype"]), (top + total.log()).view(b, heads)


def _spread(scale: torch.Tensor, rows: int, cols: int, height: int) -> torch.Tensor:
    """A scale for each element."""
    return scale.repeat_interleave(height, -2)[..., :rows, :].repeat_interleave(TILE, -1)[..., :cols]


def _linear(s: dict) -> torch.Tensor:
    x, (rows, k), n = s["x"], s["x"].shape, s["w"].shape[-2]
    height = TILE if s["x_scale"] == "block" else 1
    blocks, cols = -(-rows // height), -(-k // TILE)
    v = torch.nn.functional.pad(x.float(), (0, cols * TILE - k, 0, blocks * height - rows))
    amax = v.view(blocks, height, cols, TILE).abs().amax(dim=(1, 3))
    scale = _spread(_scale(amax, s["format"]), rows, k, height)
    x = (x.float() / scale).to(DTYPES[s["format"]]).float() * scale
    w = s["w"].float() * _spread(s["ws"], n, k, TILE)
    if s["offsets"] is None:
        return (x @ w.t()).to(s["x"].dtype)
    return torch.cat([a @ m.t() for a, m in zip(x.split(s["sizes"]), w)]).to(s["x"].dtype)


def run(state: dict):
    s = state
    if own:
        return _own(s)
    if s["op"] == "attention":
        return _attention(s)
    if s["op"] == "linear":
        return _linear(s)
    q, k = _rotated(s["q"], s), _rotated(s["k"], s)
    if s["op"] == "rope":
        return q.to(s["dtype"]), k.to(s["dtype"])
    s["keys"].flatten(0, 1)[s["slots"]] = _cached(k, s["keys"], s["cache_scale"])
    s["values"].flatten(0, 1)[s["slots"]] = _cached(s["v"].float(), s["values"], s["cache_scale"])
    return q.to(s["dtype"]), s["keys"], s["values"]


# ---------------------------------------------------------------------------
# The definitions in float64.
# ---------------------------------------------------------------------------

def _turn64(x: torch.Tensor, s: dict) -> torch.Tensor:
    """Each pair as a complex number, times factor * e^(i angle)."""
    half = s["frequencies"].numel()
    angle = s["positions"].double()[:, None, None] * s["frequencies"] * (-1.0 if s["inverse"] else 1.0)
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)
    out = x.double()
    pairs = out[..., :2 * half].unflatten(-1, (2, half) if s["layout"] == "half" else (half, 2))
    pairs = pairs.movedim(-2, -1) if s["layout"] == "half" else pairs
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    out[..., :2 * half] = (z.movedim(-1, -2) if s["layout"] == "half" else z).flatten(-2)
    return out


def _e64(q: torch.Tensor, fmt: str) -> torch.Tensor:
    """The format's nearest values, ties to even: steps of 2^(exponent - mantissa bits)."""
    mantissa, lowest = (3, -6) if fmt == "e4m3" else (2, -14)
    power = torch.frexp(q).exponent.clamp(min=lowest + 1) - 1 - mantissa
    step = torch.ldexp(torch.ones_like(q), power)
    return torch.round(q / step) * step


def _linear64(s: dict) -> torch.Tensor:
    x = s["x"].double()
    rows, k = x.shape
    height, first, out = TILE if s["x_scale"] == "block" else 1, 0, []
    values = torch.empty_like(x)
    for c in range(0, k, TILE):
        part = x[:, c:c + TILE].abs().amax(1)
        if height > 1:
            part = torch.stack([p.amax() for p in part.split(height)]).repeat_interleave(height)[:rows]
        # The format's scales and quotients are float32 values, and its codes the nearest to those:
        # neighbours of a tie go where these go.
        unit = _scale(part, s["format"]).float().double()[:, None]
        values[:, c:c + TILE] = _e64((x[:, c:c + TILE] / unit).float().double(), s["format"]) * unit
    weights, scales = (s["w"][None], s["ws"][None]) if s["offsets"] is None else (s["w"], s["ws"])
    for w, ws, count in zip(weights, scales, s["sizes"]):
        w = w.double()
        for i in range(ws.shape[0]):
            for j in range(ws.shape[1]):
                w[i * TILE:(i + 1) * TILE, j * TILE:(j + 1) * TILE] *= ws[i, j].double()
        out.append(torch.mm(values[first:first + count], w.t()))
        first += count
    return torch.cat(out)


def _attention64(s: dict):
    b, heads, dim = s["q"].shape
    page, kv = s["keys"].shape[1:3]
    out = torch.zeros((b, heads, dim), dtype=torch.float64, device="cuda")
    lse = torch.full((b, heads), -math.inf, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lengths"].tolist()):
        first = max(0, n - s["window"]) if s["window"] else 0
        if n <= first:
            continue
        at = torch.arange(first, n, device="cuda")
        where = s["table"][i, at // page], at % page
        for h in range(kv):
            k, v = (c[where[0], where[1], h].double() * s["cache_scale"] for c in (s["keys"], s["values"]))
            group = slice(h * (heads // kv), (h + 1) * (heads // kv))
            scores = torch.mm(s["q"][i, group].double(), k.t()) / math.sqrt(dim)
            lse[i, group] = torch.logsumexp(scores, -1)
            out[i, group] = torch.mm(torch.softmax(scores, -1), v)
    return out, lse


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s["op"] == "attention":
        # Launches by sequence and head: thousands of them would take too long.
        return _attention64(s) if case["sequences"] * case["kv_heads"] <= 2048 else None
    if s["op"] == "linear":
        return _linear64(s)
    q, k = _turn64(s["q"], s), _turn64(s["k"], s)
    if s["op"] == "rope":
        return q, k
    keys, values = s["keys"].double(), s["values"].double()
    fp8 = s["keys"].element_size() == 1
    for cache, rows in ((keys, k), (values, s["v"].double())):
        if fp8:
            top = torch.finfo(s["keys"].dtype).max
            rows = _e64((rows / s["cache_scale"]).clamp(-top, top), case["cache"])
        cache.flatten(0, 1)[s["slots"]] = rows
    return q, keys, values
