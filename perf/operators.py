"""Workloads of the expert and microscaled products, for timing them and comparing their outputs.

``listed()`` names the calls that a mixture-of-experts layer and a 4-bit linear
layer make of ``custom_cuda_kernals_amd.kernels``: the products grouped by
expert behind ``compute_permutation`` and ``token_gather`` (forward, and both
gradients), the MXFP4 quantiser with its inverse, and the MXFP4 product, dense
and grouped. ``draw(rng)`` gives another case of the same ranges. ``prepare``
makes a case's inputs on the GPU from a seed, ``run`` is one pass (``own``: the
package's kernels, else elementary torch operations in float32), ``exact`` is
the result in float64.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCK = 32  # elements that share an MXFP4 scale
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # |e2m1|, by code


def listed() -> list[dict]:
    return [
        # One decode step of eight sequences, top 2 of 8 experts at the width of the
        # Llama-3-8B FFN: a few rows an expert, the time is reading the weights.
        {"name": "experts_decode", "op": "linear", "tokens": 8, "top_k": 2, "experts": 8, "n": 14336, "k": 4096,
         "dtype": "bf16"},
        # Prefill of 4096 tokens through the same experts' gate projection.
        {"name": "experts_prefill", "op": "linear", "tokens": 4096, "top_k": 2, "experts": 8, "n": 14336, "k": 4096,
         "dtype": "bf16"},
        # The router benchmark's 160 experts, top 6, on narrow experts: about 77 rows each.
        {"name": "experts_many", "op": "linear", "tokens": 2048, "top_k": 6, "experts": 160, "n": 1536, "k": 2048,
         "dtype": "fp16"},
        # Odd widths, whose rows start at any element, in float32.
        {"name": "experts_odd", "op": "linear", "tokens": 333, "top_k": 3, "experts": 13, "n": 1003, "k": 777,
         "dtype": "fp32"},
        # Training: the gradient of the prefill's inputs, and a small ragged one.
        {"name": "grad_input", "op": "grad_input", "tokens": 4096, "top_k": 2, "experts": 8, "n": 14336, "k": 4096,
         "dtype": "bf16"},
        {"name": "grad_input_ragged", "op": "grad_input", "tokens": 500, "top_k": 4, "experts": 32, "n": 1412,
         "k": 1030, "dtype": "fp16"},
        # Training: the gradient of the prefill's weights, and of many narrow experts'.
        {"name": "grad_weight", "op": "grad_weight", "tokens": 4096, "top_k": 2, "experts": 8, "n": 14336, "k": 4096,
         "dtype": "bf16"},
        {"name": "grad_weight_many", "op": "grad_weight", "tokens": 1024, "top_k": 6, "experts": 64, "n": 1408,
         "k": 2048, "dtype": "fp16"},
        # A decode step's activations to MXFP4 and back: launches and latency.
        {"name": "mxfp4_few", "op": "quant", "rows": 16, "k": 4096, "dtype": "bf16"},
        # An FFN weight of the Llama-3-8B block to MXFP4 and back.
        {"name": "mxfp4_weight", "op": "quant", "rows": 14336, "k": 4096, "dtype": "bf16"},
        # A decode step of 16 sequences through an MXFP4 up projection.
        {"name": "mxfp4_decode", "op": "mxfp4", "tokens": 16, "top_k": 1, "experts": 0, "n": 14336, "k": 4096,
         "dtype": "bf16"},
        # Prefill of 4096 tokens, top 2 of 8 experts in MXFP4.
        {"name": "mxfp4_experts", "op": "mxfp4", "tokens": 4096, "top_k": 2, "experts": 8, "n": 14336, "k": 4096,
         "dtype": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng) -> int:
    """A model's width, or any number of elements."""
    if rng.random() < 0.5:
        return rng.choice([768, 1024, 1408, 1536, 2048, 2560, 4096, 5120, 7168, 8192, 14336])
    return _log_int(rng, 33, 12000)


def draw(rng) -> dict:
    op = rng.choice(["linear", "linear", "grad_input", "grad_weight", "quant", "mxfp4", "mxfp4"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "quant":
        k = _width(rng)
        return {"op": op, "rows": _log_int(rng, 1, max(1, 14336 * 4096 // k)), "k": k, "dtype": dtype}
    experts = rng.choice([8, 8, 16, 32, 64, 160, rng.randint(1, 256)])
    if op == "mxfp4" and rng.random() < 0.5:
        experts = 0
    top_k = rng.randint(1, min(8, experts)) if experts else 1
    case = {"op": op, "tokens": _log_int(rng, 1, 8192 // top_k), "top_k": top_k, "experts": experts, "n": _width(rng),
            "k": _width(rng), "dtype": dtype}
    # No more bytes of weights, and no more products, than the largest listed case has;
    # float32 products take 16 times as long.
    while max(experts, 1) * case["n"] * case["k"] * SIZES[dtype] > 2 * 8 * 14336 * 4096:
        case["n"], case["k"] = max(33, case["n"] * 2 // 3), max(33, case["k"] * 2 // 3)
    most = 8192 * 14336 * 4096 // (16 if dtype == "fp32" and op != "mxfp4" else 1)
    while case["tokens"] * top_k * case["n"] * case["k"] > most:
        case["tokens"] = case["tokens"] // 2
    return case


def _active(case: dict) -> float:
    """Experts that some token is expected to reach."""
    e = case["experts"]
    return e * (1.0 - (1.0 - case["top_k"] / e) ** case["tokens"]) if e else 1.0


def work(case: dict) -> dict:
    if case["op"] == "quant":
        m, k, size = case["rows"], case["k"], SIZES[case["dtype"]]
        blocks = -(-k // BLOCK)
        # to codes and scales, and from them to values again
        return {"bytes": 2 * m * k * size + 2 * m * blocks * (BLOCK // 2 + 1), "flops": 0}
    rows, n, k, size = case["tokens"] * case["top_k"], case["n"], case["k"], SIZES[case["dtype"]]
    flops = 2 * rows * n * k
    if case["op"] == "mxfp4":
        blocks = -(-k // BLOCK)
        return {"bytes": (rows + _active(case) * n) * blocks * (BLOCK // 2 + 1) + rows * n * size, "flops": flops}
    if case["op"] == "grad_weight":
        return {"bytes": rows * (n + k) * size + case["experts"] * n * k * size, "flops": flops}
    return {"bytes": rows * (n + k) * size + _active(case) * n * k * size, "flops": flops}


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, std: float, dtype: torch.dtype, gen: torch.Generator) -> torch.Tensor:
    return (torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen) * std).to(dtype)


def _activation(shape, dtype: torch.dtype, gen: torch.Generator) -> torch.Tensor:
    """N(0, 1) with one value in a thousand 20 times as large."""
    x = torch.randn(shape, device="cuda", dtype=torch.float32, generator=gen)
    far = torch.rand(shape, device="cuda", dtype=torch.float32, generator=gen) < 1e-3
    return torch.where(far, x * 20.0, x).to(dtype)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """MXFP4 by elementary operations: codes (two a byte, the lower element in the
    lower half, rows padded with zeros to whole blocks) and E8M0 exponent bytes."""
    k = x.shape[-1]
    blocks = -(-k // BLOCK)
    v = torch.zeros((*x.shape[:-1], blocks * BLOCK), dtype=torch.float32, device=x.device)
    v[..., :k] = x.float()
    v = v.view(*x.shape[:-1], blocks, BLOCK)
    # amax = m * 2^e with m in [0.5, 1), so floor(log2(amax)) = e - 1; the largest e2m1 exponent is 2.
    exponent = torch.frexp(v.abs().amax(-1)).exponent.to(torch.int32) - 3
    byte = (exponent + 127).clamp(0, 254)
    byte = torch.where(v.abs().amax(-1) == 0, torch.zeros_like(byte), byte)
    a = torch.ldexp(v.abs(), (127 - byte).unsqueeze(-1))
    # The code is the number of borders passed; one that is a tie goes to the even code.
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = torch.where(torch.signbit(v), code + 8, code).to(torch.uint8).flatten(-2)
    return code[..., 0::2] + code[..., 1::2] * 16, byte.to(torch.uint8)


def _values(codes: torch.Tensor, scales: torch.Tensor, k: int) -> torch.Tensor:
    """The float32 values that codes and E8M0 scales stand for."""
    half = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).to(torch.int32)
    table = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float32, device=codes.device)
    v = table[half].view(*scales.shape, BLOCK)
    scale = torch.ldexp(torch.ones_like(scales, dtype=torch.float32), scales.view(torch.uint8).to(torch.int32) - 127)
    return (v * scale.unsqueeze(-1)).flatten(-2)[..., :k]


def _routing(case: dict, gen: torch.Generator) -> tuple[torch.Tensor, list[int]]:
    """Offsets of the experts' rows, as routing gives them: some experts are liked
    more than others, and few tokens leave some without any."""
    e, t = case["experts"], case["tokens"]
    logits = torch.randn((t, e), device="cuda", generator=gen) + 0.3 * torch.randn(e, device="cuda", generator=gen)
    ids = logits.topk(case["top_k"], dim=-1).indices
    sizes = torch.bincount(ids.flatten(), minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = sizes.cumsum(0)
    return offsets, sizes.tolist()


def prepare(case: dict, seed: int) -> dict:
    gen, dtype, k = _gen(seed), DTYPES[case["dtype"]], case["k"]
    state = {"op": case["op"], "dtype": dtype, "k": k}
    if case["op"] == "quant":
        return {**state, "x": _activation((case["rows"], k), dtype, gen)}
    rows, n, e = case["tokens"] * case["top_k"], case["n"], case["experts"]
    state |= {"offsets": None, "sizes": [rows]}
    if e:
        state["offsets"], state["sizes"] = _routing(case, gen)
    if case["op"] == "mxfp4":
        codes, scales = _quantise(_activation((rows, k), torch.bfloat16, gen))
        w = [_quantise(_normal((n, k), 0.02, torch.bfloat16, gen)) for _ in range(max(e, 1))]
        w_codes, w_scales = (torch.stack(p) if e else p[0] for p in zip(*w))
        e8m0 = torch.float8_e8m0fnu
        return {**state, "x": codes, "xs": scales.view(e8m0), "w": w_codes, "ws": w_scales.view(e8m0)}
    if case["op"] != "linear":
        state["grad"] = _normal((rows, n), 0.1, dtype, gen)
    if case["op"] != "grad_input":
        state["x"] = _activation((rows, k), dtype, gen)
    if case["op"] != "grad_weight":
        state["w"] = torch.stack([_normal((n, k), 0.02, dtype, gen) for _ in range(e)])
    return state


def _own(s: dict):
    from custom_cuda_kernals_amd import kernels as K

    if s["op"] == "linear":
        return K.grouped_linear(s["x"], s["w"], s["offsets"])
    if s["op"] == "grad_input":
        return K.grouped_linear_grad_input(s["grad"], s["w"], s["offsets"])
    if s["op"] == "grad_weight":
        return K.grouped_linear_grad_weight(s["grad"], s["x"], s["offsets"])
    if s["op"] == "quant":
        codes, scales = K.mxfp4_quant(s["x"])
        return K.mxfp4_dequant(codes, scales, s["k"], s["dtype"])
    return K.mxfp4_linear(s["x"], s["xs"], s["w"], s["ws"], s["offsets"], s["dtype"])


def run(state: dict):
    s = state
    if own:
        return _own(s)
    if s["op"] == "linear":
        y = [a.float() @ w.float().t() for a, w in zip(s["x"].split(s["sizes"]), s["w"])]
        return torch.cat(y).to(s["dtype"])
    if s["op"] == "grad_input":
        return torch.cat([g.float() @ w.float() for g, w in zip(s["grad"].split(s["sizes"]), s["w"])]).to(s["dtype"])
    if s["op"] == "grad_weight":
        pairs = zip(s["grad"].split(s["sizes"]), s["x"].split(s["sizes"]))
        return torch.stack([(g.float().t() @ a.float()).to(s["dtype"]) for g, a in pairs])
    if s["op"] == "quant":
        return _values(*_quantise(s["x"]), s["k"]).to(s["dtype"])
    x = _values(s["x"], s["xs"], s["k"])
    if s["offsets"] is None:
        return (x @ _values(s["w"], s["ws"], s["k"]).t()).to(s["dtype"])
    groups = zip(x.split(s["sizes"]), s["w"], s["ws"])
    return torch.cat([a @ _values(w, ws, s["k"]).t() for a, w, ws in groups]).to(s["dtype"])


def _decode64(codes: torch.Tensor, scales: torch.Tensor, k: int) -> torch.Tensor:
    """Codes and scales in float64, from the formats' fields: (-1)^s 2^(e-1) (1 + m/2), or m/2 where e is 0."""
    c = codes.to(torch.int64)
    c = torch.stack([c % 16, c // 16], dim=-1).flatten(-2)
    sign, e, m = 1.0 - 2.0 * (c // 8).double(), (c // 2 % 4).double(), (c % 2).double()
    v = sign * torch.where(e == 0, m / 2, torch.pow(2.0, e - 1) * (1 + m / 2))
    scale = torch.pow(2.0, scales.view(torch.uint8).double() - 127)
    return (v * scale.repeat_interleave(BLOCK, dim=-1))[..., :k]


def _quant64(x: torch.Tensor) -> torch.Tensor:
    """Each block's nearest multiples, ties to the even code, in float64."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x.double(), (0, -k % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = x.abs().amax(-1, keepdim=True)
    power = torch.floor(torch.log2(torch.where(amax > 0, amax, 1.0))) - 2
    unit = torch.pow(2.0, power)
    q = (x / unit).clamp(-6, 6)
    step = torch.where(q.abs() < 2, 0.5, torch.where(q.abs() < 4, 1.0, 2.0))
    return (torch.round(q / step) * step * unit).flatten(-2)[..., :k]


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if s["op"] == "quant":
        return _quant64(s["x"])
    if s["op"] == "mxfp4":
        x, first, out = _decode64(s["x"], s["xs"], s["k"]), 0, []
        for i, rows in enumerate(s["sizes"]):
            w, ws = (s["w"], s["ws"]) if s["offsets"] is None else (s["w"][i], s["ws"][i])
            out.append(torch.mm(x[first:first + rows], _decode64(w, ws, s["k"]).t()))
            first += rows
        return torch.cat(out)
    first, out = 0, []
    for i, rows in enumerate(s["sizes"]):
        part = slice(first, first + rows)
        if s["op"] == "linear":
            out.append(torch.mm(s["x"][part].double(), s["w"][i].double().t()))
        elif s["op"] == "grad_input":
            out.append(torch.mm(s["grad"][part].double(), s["w"][i].double()))
        else:
            out.append(torch.mm(s["grad"][part].double().t(), s["x"][part].double()))
        first += rows
    return torch.stack(out) if s["op"] == "grad_weight" else torch.cat(out)
