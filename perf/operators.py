"""The operators of a talker's transformer step, the step whose tokens are the codes that the codec
decodes: the linear layers in 8-bit floating point with a scale for each block of 128, the norms
before and after a block with its gate and residual scale, rotary positions, and the penalties,
biases and grammar masks on the logits.

``prepare`` makes what a program holds before the call (everything from the seed), ``run`` is one
call: with ``own`` through ``sglang_omni_amd.kernels``, else as elementary torch operations in
float32, rounded once. ``exact`` is the same result from the definition in float64.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed() -> list[dict]:
    return [
        # the code head of one stream's decode step: one bf16 row, quantized within the call
        {"name": "linear 1x1024->2048", "op": "linear", "rows": 1, "k": 1024, "n": 2048,
         "x": "bf16", "bias": False, "out": "bf16"},
        # a layer's output projection for 64 streams, the rows already in 8 bits
        {"name": "linear 64x4096->4096", "op": "linear", "rows": 64, "k": 4096, "n": 4096,
         "x": "fp8", "bias": False, "out": "bf16"},
        # a ragged batch of utterances: rows, k and n off every tile, bias, float32 out
        {"name": "linear 773x1040->2088", "op": "linear", "rows": 773, "k": 1040, "n": 2088,
         "x": "bf16", "bias": True, "out": "f32"},
        # a long prefill's gate and up projection
        {"name": "linear 8192x4096->8192", "op": "linear", "rows": 8192, "k": 4096, "n": 8192,
         "x": "fp8", "bias": False, "out": "bf16"},
        # one stream's decode step: float32 residual, a layer scale per channel
        {"name": "norm 1x1024", "op": "norm", "rows": 1, "channels": 1024, "kind": "rms",
         "post": True, "gate": "channel", "activation": "none", "x": "f32", "y": "bf16"},
        # a conditioned block's LayerNorms: a gate per sequence, an odd width and ragged rows
        {"name": "norm 3x1001x1000", "op": "norm", "rows": 3003, "channels": 1000, "kind": "layer",
         "post": False, "gate": "sequence", "activation": "none", "x": "f16", "y": "f16"},
        # a long prefill with norms on both sides of the block and a learned gate per token
        {"name": "norm 16384x4096", "op": "norm", "rows": 16384, "channels": 4096, "kind": "rms",
         "post": True, "gate": "token", "activation": "sigmoid", "x": "bf16", "y": "bf16"},
        # 64 streams' decode step, q and k views of one qkv buffer
        {"name": "rotary 64x16+8", "op": "rotary", "tokens": 64, "heads": 16, "kv_heads": 8,
         "dim": 128, "rotary_dim": 128, "layout": "half", "scaling": "none", "start": 3000,
         "dtype": "bf16"},
        # a long context's prefill: interleaved pairs in half of each head, YaRN frequencies
        {"name": "rotary 16001x32+8", "op": "rotary", "tokens": 16001, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary_dim": 64, "layout": "interleaved", "scaling": "yarn",
         "start": 115000, "dtype": "bf16"},
        # one stream's code logits with every penalty over its last 250 codes
        {"name": "logits 1x2048", "op": "logits", "rows": 1, "vocab": 2048, "history": 250,
         "prompt": 50, "bias": 16, "allowed": "all", "dtype": "f32"},
        # 64 streams' text logits under a grammar, a long history each
        {"name": "logits 64x131072", "op": "logits", "rows": 64, "vocab": 131072, "history": 4000,
         "prompt": 1500, "bias": 100, "allowed": "some", "dtype": "f32"},
        # an odd vocabulary in bf16, most of it forbidden, short histories
        {"name": "logits 200x50257", "op": "logits", "rows": 200, "vocab": 50257, "history": 300,
         "prompt": 200, "bias": 0, "allowed": "few", "dtype": "bf16"},
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng) -> dict:
    op = rng.choice(["linear", "linear", "norm", "rotary", "logits"])
    if op == "linear":
        k = _log(rng, 8, 512) * 16
        n = _log(rng, 64, 8192)
        rows = _log(rng, 1, min(8192, 8192 * 4096 * 8192 // (k * n)))
        return {"op": op, "rows": rows, "k": k, "n": n, "x": rng.choice(["fp8", "bf16"]),
                "bias": rng.random() < 0.3, "out": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "norm":
        channels = rng.choice([_log(rng, 64, 8192), 64 * _log(rng, 2, 128)])
        x = rng.choice(["bf16", "f16", "f32"])
        gate = rng.choice(["none", "channel", "sequence", "token"])
        rows = _log(rng, 1, 16384 * 4096 // (2 * channels))
        rows = max(1, rows // 3) * 3 if gate == "sequence" else rows
        return {"op": op, "rows": rows, "channels": channels, "kind": rng.choice(["rms", "layer"]),
                "post": rng.random() < 0.6, "gate": gate,
                "activation": "none" if gate == "none" else rng.choice(["none", "sigmoid", "tanh"]),
                "x": x, "y": "bf16" if x == "f32" else x}
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 256])
        heads = rng.choice([8, 16, 32])
        kv_heads = rng.choice([1, 2, 8])
        return {"op": op, "tokens": _log(rng, 1, 16000 * 40 * 128 // ((heads + kv_heads) * dim)),
                "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary_dim": rng.choice([dim, dim // 2, 32]),
                "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["none", "linear", "yarn", "llama3"]),
                "start": _log(rng, 1, 500000), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    vocab = _log(rng, 1000, 160000)
    history = _log(rng, 1, 8000)
    return {"op": op, "rows": _log(rng, 1, min(512, 64 * 131072 // vocab)), "vocab": vocab,
            "history": history, "prompt": rng.randint(0, history),
            "bias": rng.choice([0, 16, 100]), "allowed": rng.choice(["none", "all", "some", "few"]),
            "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}


# ------------------------------------------------------------------------------ inputs


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def _blocks(rows: int, cols: int) -> tuple[int, int]:
    return -(-rows // BLOCK), -(-cols // BLOCK)


def _quantized(t, block_rows: int):
    """t's E4M3 values and the float32 scale of each block of block_rows x 128."""
    rows, cols = t.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    p = torch.zeros(rb * block_rows, cb * BLOCK, device=t.device)
    p[:rows, :cols] = t
    p = p.view(rb, block_rows, cb, BLOCK)
    amax = p.abs().amax((1, 3), keepdim=True).clamp_min(1e-12)
    q = (p * (E4M3_MAX / amax)).view(rb * block_rows, cb * BLOCK)[:rows, :cols]
    return q.contiguous().to(torch.float8_e4m3fn), (amax / E4M3_MAX).view(rb, cb)


def prepare(case: dict, seed: int) -> SimpleNamespace:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return SimpleNamespace(case=case, **globals()["_prepare_" + case["op"]](case, g))


def _prepare_linear(case, g) -> dict:
    rows, k, n = case["rows"], case["k"], case["n"]
    # a layer's input after its norm: near unit variance, some channels much larger
    x = _randn(g, rows, k) * torch.exp(_randn(g, k, std=0.7))
    weight, weight_scale = _quantized(_randn(g, n, k, std=k ** -0.5), BLOCK)
    s = {"weight": weight, "weight_scale": weight_scale,
         "bias": _randn(g, n, std=0.1) if case["bias"] else None, "x_scale": None}
    if case["x"] == "fp8":
        s["x"], s["x_scale"] = _quantized(x, 1)
    else:
        s["x"] = x.to(torch.bfloat16)
    return s


def _prepare_norm(case, g) -> dict:
    rows, c = case["rows"], case["channels"]
    s = {"x": _randn(g, rows, c, std=2.0).to(DTYPES[case["x"]]),
         "y": (_randn(g, rows, c) + 0.1).to(DTYPES[case["y"]]),
         "pre_weight": 1 + _randn(g, c, std=0.1), "pre_bias": None,
         "post_weight": 1 + _randn(g, c, std=0.1) if case["post"] else None, "post_bias": None}
    if case["kind"] == "layer":
        s["pre_bias"] = _randn(g, c, std=0.1)
        s["post_bias"] = _randn(g, c, std=0.1) if case["post"] else None
    gates = {"none": 0, "channel": 1, "sequence": 3, "token": rows}[case["gate"]]
    dtype = torch.float32 if case["gate"] == "channel" else DTYPES[case["y"]]
    s["gate"] = _randn(g, gates, c).to(dtype) if gates else None
    s["scale"] = 0.7
    s["eps"] = 1e-5
    return s


def _prepare_rotary(case, g) -> dict:
    t, h, kh, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    qkv = _randn(g, t, (h + 2 * kh) * d).to(DTYPES[case["dtype"]])
    positions = torch.arange(t, device="cuda") + case["start"]
    if t <= 512:  # a decode batch: each token at its own stream's position
        positions = torch.randint(0, case["start"] + 1, (t,), generator=g, device="cuda")
    inv_freq, factor = _frequencies(case["rotary_dim"], case["scaling"])
    return {"q": qkv[:, :h * d].view(t, h, d), "k": qkv[:, h * d:(h + kh) * d].view(t, kh, d),
            "positions": positions, "inv_freq": inv_freq.to("cuda"), "factor": factor}


def _frequencies(dim: int, scaling: str) -> tuple[torch.Tensor, float]:
    """The radians per position of each pair, float64, and the factor on cos and sin."""
    base, original, factor = 1e6, 8192, 16.0
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "none":
        return inv, 1.0
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "llama3":
        # wavelengths longer than the original context are divided by the factor, those shorter
        # than a quarter of it kept, between them a blend
        turns = original * inv / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return inv * (keep + (1 - keep) / factor), 1.0
    # YaRN: pairs that turn fewer than once in the original context are divided by the factor,
    # those that turn more than 32 times kept, a ramp over the pair index between them
    def pair(turns):
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
    low, high = max(math.floor(pair(32)), 0), min(math.ceil(pair(1)), dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
    return inv * (1 - ramp) + inv / factor * ramp, 0.1 * math.log(factor) + 1.0


def _prepare_logits(case, g) -> dict:
    rows, v, h = case["rows"], case["vocab"], case["history"]
    logits = _randn(g, rows, v, std=3.0)
    # recent tokens repeat: a skewed distribution over the vocabulary, each row its own length
    u = torch.rand(rows, h, generator=g, device="cuda")
    s = {"logits": logits.to(DTYPES[case["dtype"]]),
         "history": (u.pow(3) * v).long().clamp_max(v - 1).to(torch.int32),
         "lengths": torch.randint(h // 2, h + 1, (rows,), generator=g, device="cuda",
                                  dtype=torch.int32)}
    s["prompt_lengths"] = s["lengths"].clamp_max(case["prompt"])
    s["repetition"] = 1 + 0.3 * torch.rand(rows, generator=g, device="cuda")
    s["frequency"] = 0.2 * torch.rand(rows, generator=g, device="cuda")
    s["presence"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
    s["bias_tokens"] = s["bias_values"] = s["allowed"] = None
    if case["bias"]:
        s["bias_tokens"] = torch.rand(rows, v, generator=g, device="cuda").topk(
            min(case["bias"], v), dim=1).indices.to(torch.int32)
        s["bias_values"] = _randn(g, *s["bias_tokens"].shape, std=4.0)
    if case["allowed"] != "none":
        words = -(-v // 32)
        bits = torch.randint(-2**31, 2**31, (rows, words), generator=g, device="cuda")
        if case["allowed"] == "all":
            bits = torch.full_like(bits, -1)
        elif case["allowed"] == "few":
            bits = torch.where(torch.rand(rows, words, generator=g, device="cuda") < 0.01, bits, 0)
        s["allowed"] = bits.to(torch.int32)
    return s


# ------------------------------------------------------------------------------ one call


def run(s: SimpleNamespace):
    if own:
        return globals()["_own_" + s.case["op"]](_kernels(), s)
    return globals()["_plain_" + s.case["op"]](s)


def _kernels():
    """The framework's kernels, imported where they are called."""
    package = str(Path.cwd() / "sglang-omni_amd")
    if package not in sys.path:
        sys.path.insert(1, package)
    from sglang_omni_amd import kernels

    return kernels


def _own_linear(kernels, s):
    weight = kernels.BlockFp8Weight(s.weight, s.weight_scale, s.bias)
    x = s.x if s.x_scale is None else kernels.BlockFp8Rows(s.x, s.x_scale)
    return kernels.block_fp8_linear(x, weight, out_dtype=DTYPES[s.case["out"]])


def _own_norm(kernels, s):
    return kernels.gated_residual_norm(
        s.x, s.y, norm=s.case["kind"], eps=s.eps, post_norm=s.case["post"],
        post_weight=s.post_weight, post_bias=s.post_bias, pre_weight=s.pre_weight,
        pre_bias=s.pre_bias, gate=s.gate, gate_activation=s.case["activation"], scale=s.scale,
        normed_dtype=s.y.dtype)


def _own_rotary(kernels, s):
    return kernels.apply_rotary(s.q, s.k, s.positions, s.inv_freq, layout=s.case["layout"],
                                factor=s.factor)


def _own_logits(kernels, s):
    return kernels.adjust_logits(
        s.logits, history=s.history, lengths=s.lengths, prompt_lengths=s.prompt_lengths,
        repetition=s.repetition, frequency=s.frequency, presence=s.presence,
        bias_tokens=s.bias_tokens, bias_values=s.bias_values, allowed=s.allowed)


def _dequantized(q, scale, block_rows: int):
    rows, cols = q.shape
    full = scale.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return q.float() * full


def _plain_linear(s):
    x = s.x
    if s.x_scale is None:
        # each row's groups of 128: the largest magnitude to 448, one rounding to E4M3
        rows, k = x.shape
        p = torch.nn.functional.pad(x.float(), (0, -k % BLOCK)).view(rows, -1, BLOCK)
        amax = p.abs().amax(2, keepdim=True)
        tiny, most = amax < 2.0 ** -100, torch.full_like(amax, E4M3_MAX)
        q = p * torch.where(tiny, 1.0, most / amax)
        q = q.view(rows, -1)[:, :k].to(torch.float8_e4m3fn)
        x = _dequantized(q, torch.where(tiny, 1.0, amax / most)[..., 0], 1)
    else:
        x = _dequantized(x, s.x_scale, 1)
    y = x @ _dequantized(s.weight, s.weight_scale, BLOCK).T
    if s.bias is not None:
        y = y + s.bias
    return y.to(DTYPES[s.case["out"]])


def _norm(v, kind: str, eps: float, weight, bias):
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    if weight is not None:
        v = v * weight
    return v if bias is None else v + bias


def _gate(gate, rows: int, activation: str):
    gate = {"none": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[activation](gate)
    return gate.repeat_interleave(rows // gate.shape[0], 0)


def _plain_norm(s):
    y = s.y.float()
    if s.case["post"]:
        y = _norm(y, s.case["kind"], s.eps, s.post_weight, s.post_bias)
    if s.gate is not None:
        y = y * _gate(s.gate.float(), y.shape[0], s.case["activation"])
    h = s.x.float() + s.scale * y
    normed = _norm(h, s.case["kind"], s.eps, s.pre_weight, s.pre_bias)
    return h.to(s.x.dtype), normed.to(s.y.dtype)


def _turned(t, cos, sin, layout: str):
    """t [tokens, heads, dim] with its first 2 * pairs values turned, in cos's type."""
    pairs = cos.shape[1]
    cos, sin = cos[:, None], sin[:, None]
    v = t.to(cos.dtype)
    a, b = ((v[..., :pairs], v[..., pairs:2 * pairs]) if layout == "half" else
            (v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]))
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, v[..., 2 * pairs:]], -1)


def _plain_rotary(s):
    # the angles alone in 64 bits: at position 100 000 a float32 angle is 0.004 off, as much as a
    # bf16 rounding
    angle = s.positions.double()[:, None] * s.inv_freq
    cos, sin = (angle.cos() * s.factor).float(), (angle.sin() * s.factor).float()
    return tuple(_turned(t, cos, sin, s.case["layout"]).to(t.dtype) for t in (s.q, s.k))


def _plain_logits(s):
    v = s.logits.float()
    rows, vocab = v.shape
    at = torch.arange(s.history.shape[1], device=v.device)
    tokens = s.history.long()
    held = (at < s.lengths[:, None]).float()
    made = held * (at >= s.prompt_lengths[:, None])
    seen = torch.zeros_like(v).scatter_add_(1, tokens, held) > 0
    count = torch.zeros_like(v).scatter_add_(1, tokens, made)
    repeated = torch.where(v > 0, v / s.repetition[:, None], v * s.repetition[:, None])
    v = torch.where(seen, repeated, v)
    v = v - s.frequency[:, None] * count - s.presence[:, None] * (count > 0)
    if s.bias_tokens is not None:
        v = v.scatter_add(1, s.bias_tokens.long(), s.bias_values)
    if s.allowed is not None:
        token = torch.arange(vocab, device=v.device)
        bit = (s.allowed[:, token // 32] >> (token % 32).to(torch.int32)) & 1
        v = torch.where(bit > 0, v, -math.inf)
    return v.to(s.logits.dtype)


# ------------------------------------------------------------------------------ float64


def exact(case: dict, seed: int):
    return globals()["_exact_" + case["op"]](case, prepare(case, seed))


def _expand(scale, per_row: int, rows: int, cols: int):
    r = torch.arange(rows, device=scale.device) // per_row
    c = torch.arange(cols, device=scale.device) // BLOCK
    return scale.double()[r][:, c]


def _exact_linear(case, s):
    rows, k, n = case["rows"], case["k"], case["n"]
    if s.x_scale is None:
        x = s.x.double()
        group = torch.arange(k, device=x.device) // BLOCK
        amax = torch.zeros(rows, _blocks(1, k)[1], dtype=torch.float64, device=x.device)
        amax = amax.scatter_reduce(1, group.expand(rows, k), x.abs(), "amax")[:, group]
        # the operator's 8-bit values are part of its definition: one float32 product each
        unit = (torch.tensor(E4M3_MAX, device=x.device) / amax.float())
        unit = torch.where(amax < 2.0 ** -100, torch.ones_like(unit), unit)
        back = torch.where(amax < 2.0 ** -100, torch.ones_like(amax), amax / E4M3_MAX)
        x = (s.x.float() * unit).to(torch.float8_e4m3fn).double() * back
    else:
        x = s.x.double() * _expand(s.x_scale, 1, rows, k)
    y = torch.matmul(x, (s.weight.double() * _expand(s.weight_scale, BLOCK, n, k)).t())
    return y if s.bias is None else y + s.bias.double()


def _exact_norm(case, s):
    rows, c = s.y.shape

    def norm(v, weight, bias):
        mean = v.sum(1, keepdim=True) / c if case["kind"] == "layer" else 0.0
        var = ((v - mean) ** 2).sum(1, keepdim=True) / c
        v = (v - mean) * (var + s.eps) ** -0.5
        v = v if weight is None else v * weight.double()
        return v if bias is None else v + bias.double()

    u = s.y.double()
    if case["post"]:
        u = norm(u, s.post_weight, s.post_bias)
    if s.gate is not None:
        z = s.gate.double()
        if case["activation"] == "sigmoid":
            z = 1 / (1 + torch.exp(-z))
        elif case["activation"] == "tanh":
            z = torch.expm1(2 * z) / (torch.expm1(2 * z) + 2)
        u = u * z[torch.arange(rows, device=u.device) // (rows // z.shape[0])]
    h = s.x.double() + s.scale * u
    return h, norm(h, s.pre_weight, s.pre_bias)


def _exact_rotary(case, s):
    pairs = case["rotary_dim"] // 2
    angle = torch.outer(s.positions.double(), s.inv_freq)
    turn = torch.polar(torch.full_like(angle, s.factor), angle)[:, None]
    outputs = []
    for t in (s.q, s.k):
        v = t.double().clone()
        i = torch.arange(pairs, device=v.device)
        first, second = (i, i + pairs) if case["layout"] == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(v[..., first], v[..., second]) * turn
        v[..., first], v[..., second] = z.real, z.imag
        outputs.append(v)
    return tuple(outputs)


def _exact_logits(case, s):
    v = s.logits.double()
    vocab = case["vocab"]
    for row in range(case["rows"]):
        length, prompt = int(s.lengths[row]), int(s.prompt_lengths[row])
        tokens = s.history[row, :length].long()
        seen = torch.unique(tokens)
        old = v[row, seen]
        r = s.repetition[row].double()
        v[row, seen] = torch.where(old > 0, old / r, old * r)
        count = torch.bincount(tokens[prompt:], minlength=vocab).double()
        v[row] -= s.frequency[row].double() * count
        v[row] -= s.presence[row].double() * (count != 0)
        if s.bias_tokens is not None:
            v[row, s.bias_tokens[row].long()] += s.bias_values[row].double()
    if s.allowed is not None:
        shifts = torch.arange(32, dtype=torch.int32, device=v.device)
        bits = ((s.allowed[:, :, None] >> shifts) & 1).view(case["rows"], -1)[:, :vocab]
        v[bits == 0] = -math.inf
    return v


# ------------------------------------------------------------------------------ work


def work(case: dict) -> dict:
    return globals()["_work_" + case["op"]](case)


def _size(name: str) -> int:
    return 4 if name == "f32" else 2


def _work_linear(case):
    rows, k, n = case["rows"], case["k"], case["n"]
    wr, kb = _blocks(n, k)
    x = rows * k * 2 if case["x"] == "bf16" else rows * (k + 4 * kb)
    return {"bytes": x + n * k + 4 * wr * kb + (4 * n if case["bias"] else 0)
            + rows * n * _size(case["out"]), "flops": 2 * rows * n * k}


def _work_norm(case):
    rows, c = case["rows"], case["channels"]
    gates = {"none": 0, "channel": 1, "sequence": 3, "token": rows}[case["gate"]]
    gate = gates * c * (4 if case["gate"] == "channel" else _size(case["y"]))
    vectors = (1 + case["post"]) * (2 if case["kind"] == "layer" else 1) * c * 4
    return {"bytes": rows * c * 2 * (_size(case["x"]) + _size(case["y"])) + gate + vectors,
            "flops": rows * c * (14 if case["post"] else 8)}


def _work_rotary(case):
    t, heads, d = case["tokens"], case["heads"] + case["kv_heads"], case["dim"]
    return {"bytes": t * heads * d * 2 * _size(case["dtype"]) + t * 8 + case["rotary_dim"] * 4,
            "flops": t * (heads * 3 * case["rotary_dim"] + 10 * case["rotary_dim"])}


def _work_logits(case):
    rows, v = case["rows"], case["vocab"]
    mask = 0 if case["allowed"] == "none" else -(-v // 32) * 4
    return {"bytes": rows * (v * 2 * _size(case["dtype"]) + mask + case["history"] * 3
                             + case["bias"] * 8 + 20), "flops": rows * v * 4}
