"""The operators of a talker's attention over its whole context: the norms and rotary positions of
the query and key heads, the paged key-value cache with its 8-bit rows, the attention of whole prompts
and the attention of one new token over the cache.

``prepare`` makes what a program holds before the call (everything from the seed), ``run`` is one
call: with ``own`` through ``sglang_omni_amd.kernels``, else as elementary torch operations in
float32, rounded once. ``exact`` is the same result from the definition in float64.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path
from types import SimpleNamespace

import torch

own = False

E4M3_MAX = 448.0
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32,
          "e4m3": torch.float8_e4m3fn}


def listed() -> list[dict]:
    return [
        # 64 streams' decode step: q, k and v views of one qkv buffer, k and v into the cache
        {"name": "heads 64x16+8 cached", "op": "heads", "tokens": 64, "heads": 16, "kv_heads": 8,
         "dim": 128, "rotary_dim": 128, "layout": "half", "cached": True, "page": 16,
         "dtype": "bf16"},
        # a long prompt's heads, an odd number of tokens
        {"name": "heads 16001x32+8", "op": "heads", "tokens": 16001, "heads": 32, "kv_heads": 8,
         "dim": 128, "rotary_dim": 128, "layout": "half", "cached": False, "page": 0,
         "dtype": "bf16"},
        # a step's rows to an 8-bit cache and back
        {"name": "cache 64x8x128 e4m3", "op": "cache", "tokens": 64, "kv_heads": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "held": "e4m3"},
        # a long prompt's rows to an 8-bit cache of larger pages, and back for its next piece
        {"name": "cache 30011x8x128 e4m3", "op": "cache", "tokens": 30011, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "held": "e4m3"},
        # one short utterance
        {"name": "prompt 37", "op": "prompt", "batch": 1, "longest": 37, "ragged": False,
         "before": 0, "heads": 16, "kv_heads": 8, "dim": 128, "causal": True, "dtype": "bf16"},
        # a packed batch of utterances of their own lengths, seven query heads to a key head
        {"name": "prompt 24 ragged to 700", "op": "prompt", "batch": 24, "longest": 700,
         "ragged": True, "before": 0, "heads": 14, "kv_heads": 2, "dim": 64, "causal": True,
         "dtype": "f16"},
        # the next piece of a long prompt, over the keys of what came before
        {"name": "prompt 500 after 20000", "op": "prompt", "batch": 1, "longest": 500,
         "ragged": False, "before": 20000, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True,
         "dtype": "bf16"},
        # a whole long prompt
        {"name": "prompt 16384", "op": "prompt", "batch": 1, "longest": 16384, "ragged": False,
         "before": 0, "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "dtype": "bf16"},
        # one stream's next token, early in its context
        {"name": "decode 1x300", "op": "decode", "batch": 1, "longest": 300, "ragged": False,
         "heads": 16, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16", "held": "bf16"},
        # 64 streams' next tokens, each at its own length
        {"name": "decode 64 ragged to 5000", "op": "decode", "batch": 64, "longest": 5000,
         "ragged": True, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "bf16",
         "held": "bf16"},
        # a few streams with an odd grouping, small heads and half precision
        {"name": "decode 9 ragged to 20000", "op": "decode", "batch": 9, "longest": 20000,
         "ragged": True, "heads": 14, "kv_heads": 2, "dim": 64, "page": 32, "dtype": "f16",
         "held": "f16"},
        # two streams with very long contexts in an 8-bit cache
        {"name": "decode 2x131072 e4m3", "op": "decode", "batch": 2, "longest": 131072,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16",
         "held": "e4m3"},
    ]


def _log(rng, low: int, high: int) -> int:
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


HEADS = [(8, 8), (16, 8), (16, 2), (32, 8), (14, 2), (24, 3), (20, 1)]


def draw(rng) -> dict:
    op = rng.choice(["heads", "cache", "prompt", "prompt", "decode", "decode"])
    heads, kv_heads = rng.choice(HEADS)
    dim = rng.choice([64, 80, 128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "heads":
        return {"op": op, "tokens": _log(rng, 1, 16000 * 40 * 128 // ((heads + 2 * kv_heads) * dim)),
                "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotary_dim": rng.choice([dim, dim, dim // 2]),
                "layout": rng.choice(["half", "interleaved"]), "cached": rng.random() < 0.5,
                "page": rng.choice([1, 16, 24, 64]),
                "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    if op == "cache":
        return {"op": op, "tokens": _log(rng, 1, 30000 * 8 * 128 // (kv_heads * dim)),
                "kv_heads": kv_heads, "dim": dim, "page": rng.choice([1, 16, 24, 64]),
                "dtype": dtype, "held": rng.choice(["e4m3", "e4m3", dtype])}
    if op == "prompt":
        # pairs of a query and a key, over the heads, at most those of the largest listed case
        pairs = 16384 * 16384 // 2 * 32 * 128 // (heads * dim)
        batch = rng.choice([1, 1, _log(rng, 2, 64)])
        longest = _log(rng, 1, min(16384, math.isqrt(pairs // batch)))
        before = rng.choice([0, 0, _log(rng, 1, min(20000, max(1, pairs // (2 * batch * longest))))])
        return {"op": op, "batch": batch, "longest": longest, "ragged": batch > 1,
                "before": before, "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "causal": rng.random() < 0.8, "dtype": dtype}
    held = rng.choice([dtype, dtype, "e4m3"])
    rows = 262144 * 8 * 128 // (kv_heads * dim * (1 if held == "e4m3" else 2))
    batch = _log(rng, 1, 128)
    longest = _log(rng, 1, min(131072, rows // batch))
    return {"op": op, "batch": batch, "longest": longest, "ragged": rng.random() < 0.6,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": rng.choice([1, 16, 24, 64]),
            "dtype": dtype, "held": held}


def _lengths(case: dict) -> list[int]:
    """The sequences' lengths: all the longest, or spread between one and it, one as long as it."""
    batch, longest = case["batch"], case["longest"]
    if not case["ragged"]:
        return [longest] * batch
    rng = random.Random(batch * 1000003 + longest)
    return [longest] + [rng.randint(1, longest) for _ in range(batch - 1)]


# ------------------------------------------------------------------------------ inputs


def _randn(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda") * std


def prepare(case: dict, seed: int) -> SimpleNamespace:
    g = torch.Generator(device="cuda").manual_seed(seed)
    return SimpleNamespace(case=case, **globals()["_prepare_" + case["op"]](case, g))


def _cache(case, pages: int, g, held: str) -> dict:
    """An empty cache [pages, kv_heads, page, dim]."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    s = {"keys": torch.zeros(shape, device="cuda", dtype=torch.float32).to(DTYPES[held]),
         "values": torch.zeros(shape, device="cuda", dtype=torch.float32).to(DTYPES[held]),
         "key_scale": None, "value_scale": None}
    if held == "e4m3":
        s["key_scale"] = torch.ones(shape[:3], device="cuda")
        s["value_scale"] = torch.ones(shape[:3], device="cuda")
    return s


def _prepare_heads(case, g) -> dict:
    t, h, kh, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    qkv = _randn(g, t, (h + 2 * kh) * d, std=2.0).to(DTYPES[case["dtype"]])
    positions = torch.arange(t, device="cuda") + 3000
    if t <= 512:  # a decode batch: each token at its own stream's position
        positions = torch.randint(0, 30000, (t,), generator=g, device="cuda")
    i = torch.arange(0, case["rotary_dim"], 2, dtype=torch.float64, device="cuda")
    s = {"q": qkv[:, :h * d].view(t, h, d), "k": qkv[:, h * d:(h + kh) * d].view(t, kh, d),
         "v": qkv[:, (h + kh) * d:].view(t, kh, d), "positions": positions,
         "inv_freq": 1e6 ** (-i / case["rotary_dim"]),
         "q_weight": 1 + _randn(g, d, std=0.2), "k_weight": 1 + _randn(g, d, std=0.2)}
    if case["cached"]:
        pages = -(-t // case["page"]) + 3
        s.update(_cache(case, pages, g, "bf16" if case["dtype"] == "f32" else case["dtype"]))
        s["slots"] = torch.randperm(pages * case["page"], generator=g, device="cuda")[:t]
    return s


def _prepare_cache(case, g) -> dict:
    t, kh, d = case["tokens"], case["kv_heads"], case["dim"]
    kv = _randn(g, t, 2 * kh * d).to(DTYPES[case["dtype"]])
    pages = -(-t // case["page"]) + 3
    # pages in any order, the tokens of a page side by side
    order = torch.randperm(pages, generator=g, device="cuda")
    at = torch.arange(t, device="cuda")
    return {"k": kv[:, :kh * d].view(t, kh, d), "v": kv[:, kh * d:].view(t, kh, d),
            "slots": order[at // case["page"]] * case["page"] + at % case["page"],
            **_cache(case, pages, g, case["held"])}


def _starts(lengths) -> torch.Tensor:
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def _prepare_prompt(case, g) -> dict:
    h, kh, d = case["heads"], case["kv_heads"], case["dim"]
    lengths = _lengths(case)
    key_lengths = [n + case["before"] for n in lengths]
    dtype = DTYPES[case["dtype"]]
    # normed heads: rows of length sqrt(dim), some queries that look sharply at a few keys
    q = _randn(g, sum(lengths), h, d) * torch.exp(_randn(g, sum(lengths), h, 1, std=0.5))
    k = _randn(g, sum(key_lengths), kh, d)
    v = _randn(g, sum(key_lengths), kh, d)
    return {"q": q.to(dtype), "k": k.to(dtype), "v": v.to(dtype), "starts": _starts(lengths),
            "key_starts": _starts(key_lengths), "scale": d ** -0.5}


def _prepare_decode(case, g) -> dict:
    b, h, kh, d, page = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "page"))
    lengths = _lengths(case)
    counts = [-(-n // page) for n in lengths]
    pages = sum(counts) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(b, max(counts), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(counts):
        table[i, :n] = order[at:at + n]
        at += n
    s = _cache(case, 1, g, case["held"])
    shape = (pages, kh, page, d)
    for name in ("keys", "values"):
        x = _randn(g, *shape)
        if case["held"] == "e4m3":
            amax = x.abs().amax(3, keepdim=True)
            s[name[:-1] + "_scale"] = (amax / E4M3_MAX)[..., 0]
            x = x * (E4M3_MAX / amax)
        s[name] = x.to(DTYPES[case["held"]])
        del x
    q = _randn(g, b, h, d) * torch.exp(_randn(g, b, h, 1, std=0.5))
    return {**s, "q": q.to(DTYPES[case["dtype"]]), "table": table, "scale": d ** -0.5,
            "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
            "host_lengths": lengths}


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


def _own_cache_of(kernels, s):
    return kernels.PagedKvCache(s.keys, s.values, s.key_scale, s.value_scale)


def _own_heads(kernels, s):
    cached = {}
    if s.case["cached"]:
        cached = {"v": s.v, "cache": _own_cache_of(kernels, s), "slots": s.slots}
    q, k = kernels.norm_rotary(s.q, s.k, s.positions, s.inv_freq, q_weight=s.q_weight,
                               k_weight=s.k_weight, eps=EPS, layout=s.case["layout"], **cached)
    return (q, k, s.keys, s.values) if cached else (q, k)


def _own_cache(kernels, s):
    cache = _own_cache_of(kernels, s)
    kernels.write_kv_cache(cache, s.k, s.v, s.slots)
    return kernels.read_kv_cache(cache, s.slots, dtype=s.k.dtype)


def _own_prompt(kernels, s):
    return kernels.prompt_attention(s.q, s.k, s.v, s.starts, key_starts=s.key_starts,
                                    causal=s.case["causal"], scale=s.scale)


def _own_decode(kernels, s):
    return kernels.paged_attention(s.q, _own_cache_of(kernels, s), s.table, s.lengths, scale=s.scale)


def _rows(held, slots, page: int):
    """The rows [tokens, kv_heads, ...] of a cache at slots."""
    return held[slots // page, :, slots % page]


def _put(held, slots, page: int, rows) -> None:
    held[slots // page, :, slots % page] = rows


def _plain_heads(s):
    # the angles alone in 64 bits: at far positions a float32 angle is as far off as a bf16 rounding
    angle = s.positions.double()[:, None] * s.inv_freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    pairs = cos.shape[2]
    outputs = []
    for t, weight in ((s.q, s.q_weight), (s.k, s.k_weight)):
        v = t.float()
        v = v / torch.sqrt((v * v).mean(2, keepdim=True) + EPS) * weight
        if s.case["layout"] == "half":
            a, b = v[..., :pairs], v[..., pairs:2 * pairs]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = v[..., 0:2 * pairs:2], v[..., 1:2 * pairs:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        outputs.append(torch.cat([turned, v[..., 2 * pairs:]], -1).to(t.dtype))
    if s.case["cached"]:
        _put(s.keys, s.slots, s.case["page"], outputs[1].to(s.keys.dtype))
        _put(s.values, s.slots, s.case["page"], s.v.to(s.values.dtype))
        outputs += [s.keys, s.values]
    return tuple(outputs)


def _plain_cache(s):
    page = s.case["page"]
    outputs = []
    for rows, held, scales in ((s.k, s.keys, s.key_scale), (s.v, s.values, s.value_scale)):
        if scales is None:
            _put(held, s.slots, page, rows.to(held.dtype))
            outputs.append(_rows(held, s.slots, page).to(rows.dtype))
            continue
        x = rows.float()
        amax = x.abs().amax(2, keepdim=True)
        tiny, most = amax < 2.0 ** -100, torch.full_like(amax, E4M3_MAX)
        scale = torch.where(tiny, 1.0, amax / most)
        q = (x * torch.where(tiny, 1.0, most / amax)).to(torch.float8_e4m3fn)
        # bytes are moved: 8-bit floats have no indexing
        _put(held.view(torch.uint8), s.slots, page, q.view(torch.uint8))
        _put(scales, s.slots, page, scale[..., 0])
        back = _rows(held.view(torch.uint8), s.slots, page).view(torch.float8_e4m3fn)
        outputs.append((back.float() * _rows(scales, s.slots, page)[..., None]).to(rows.dtype))
    return tuple(outputs)


def _softmax(scores):
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    return p / p.sum(-1, keepdim=True)


def _plain_prompt(s):
    group = s.case["heads"] // s.case["kv_heads"]
    out = torch.empty_like(s.q)
    lengths = _lengths(s.case)
    first = first_key = 0
    for n in lengths:
        m = n + s.case["before"]
        q = s.q[first:first + n].float().transpose(0, 1)
        k = s.k[first_key:first_key + m].float().transpose(0, 1)
        v = s.v[first_key:first_key + m].float().transpose(0, 1)
        hidden = None
        if s.case["causal"]:
            at = torch.arange(m, device=q.device)
            hidden = at[None, :] > at[m - n:, None]
        # some key heads at a time: their scores stay under 4 GiB
        step = max(1, 2 ** 30 // (group * n * m))
        for j in range(0, s.case["kv_heads"], step):
            kj, vj = k[j:j + step, None], v[j:j + step, None]
            qj = q[j * group:(j + kj.shape[0]) * group].unflatten(0, (-1, group))
            scores = torch.matmul(qj, kj.transpose(2, 3)) * s.scale
            if hidden is not None:
                scores.masked_fill_(hidden, -math.inf)
            o = torch.matmul(_softmax(scores), vj).flatten(0, 1)
            out[first:first + n, j * group:j * group + o.shape[0]] = o.transpose(0, 1).to(out.dtype)
        first, first_key = first + n, first_key + m
    return out


def _dense(held, scales, pages, length: int):
    """A sequence's rows [kv_heads, length, dim] in float32."""
    if scales is not None:
        x = held.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * scales[pages][..., None]
    else:
        x = held[pages].float()
    return x.transpose(0, 1).flatten(1, 2)[:, :length]


def _plain_decode(s):
    group = s.case["heads"] // s.case["kv_heads"]
    out = torch.empty_like(s.q)
    for i, n in enumerate(s.host_lengths):
        pages = s.table[i, :-(-n // s.case["page"])].long()
        k = _dense(s.keys, s.key_scale, pages, n)
        v = _dense(s.values, s.value_scale, pages, n)
        q = s.q[i].float().unflatten(0, (-1, group))
        p = _softmax(torch.matmul(q, k.transpose(1, 2)) * s.scale)
        out[i] = torch.matmul(p, v).flatten(0, 1).to(out.dtype)
    return out


# ------------------------------------------------------------------------------ float64


def exact(case: dict, seed: int):
    return globals()["_exact_" + case["op"]](case, prepare(case, seed))


def _exact_heads(case, s):
    pairs = case["rotary_dim"] // 2
    i = torch.arange(pairs, device="cuda")
    first, second = (i, i + pairs) if case["layout"] == "half" else (2 * i, 2 * i + 1)
    angle = torch.outer(s.positions.double(), s.inv_freq)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    outputs = []
    for t, weight in ((s.q, s.q_weight), (s.k, s.k_weight)):
        v = t.double()
        v = v * ((v ** 2).sum(2, keepdim=True) / case["dim"] + EPS) ** -0.5 * weight.double()
        z = torch.complex(v[..., first], v[..., second]) * turn
        v[..., first], v[..., second] = z.real, z.imag
        outputs.append(v)
    if case["cached"]:
        for held, rows in ((s.keys, outputs[1]), (s.values, s.v.double())):
            held = held.double().transpose(1, 2).flatten(0, 1).index_copy(0, s.slots, rows)
            outputs.append(held.unflatten(0, (-1, case["page"])).transpose(1, 2))
    return tuple(outputs)


def _exact_cache(case, s):
    if case["held"] != "e4m3":
        return s.k.double(), s.v.double()
    outputs = []
    for rows in (s.k, s.v):
        x = rows.double()
        amax = torch.linalg.vector_norm(x, math.inf, dim=2, keepdim=True)
        # the 8-bit values are part of the definition: one float32 quotient and product each
        unit = torch.tensor(E4M3_MAX, device="cuda") / amax.float()
        tiny = amax < 2.0 ** -100
        q = (rows.float() * torch.where(tiny, torch.ones_like(unit), unit)).to(torch.float8_e4m3fn)
        outputs.append(q.double() * torch.where(tiny, torch.ones_like(amax), amax / E4M3_MAX))
    return tuple(outputs)


def _exact_prompt(case, s):
    heads, group = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    starts, key_starts = s.starts.tolist(), s.key_starts.tolist()
    for b in range(case["batch"]):
        q0, q1, k0, k1 = *starts[b:b + 2], *key_starts[b:b + 2]
        after = torch.ones(q1 - q0, k1 - k0, dtype=torch.bool, device="cuda").triu(
            (k1 - k0) - (q1 - q0) + 1) if case["causal"] else None
        for h in range(heads):
            k = s.k[k0:k1, h // group].double().contiguous()
            scores = (s.q[q0:q1, h].double() * s.scale).mm(k.t())
            if after is not None:
                scores[after] = -math.inf
            scores -= torch.logsumexp(scores, 1, keepdim=True)
            out[q0:q1, h] = scores.exp_().mm(s.v[k0:k1, h // group].double())
    return out


def _exact_decode(case, s):
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.empty(s.q.shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(s.lengths.tolist()):
        at = torch.arange(n, device="cuda")
        pages, offset = s.table[b].long()[at // page], at % page
        for j in range(case["kv_heads"]):
            if case["held"] == "e4m3":
                k, v = (t.view(torch.uint8)[pages, j, offset].view(torch.float8_e4m3fn).double()
                        * scale[pages, j, offset].double()[:, None]
                        for t, scale in ((s.keys, s.key_scale), (s.values, s.value_scale)))
            else:
                k, v = s.keys[pages, j, offset].double(), s.values[pages, j, offset].double()
            scores = (s.q[b, j * group:(j + 1) * group].double() * s.scale).mm(k.t())
            out[b, j * group:(j + 1) * group] = (
                scores - torch.logsumexp(scores, 1, keepdim=True)).exp().mm(v)
    return out


# ------------------------------------------------------------------------------ work


def work(case: dict) -> dict:
    return globals()["_work_" + case["op"]](case)


def _size(name: str) -> int:
    return {"f32": 4, "e4m3": 1}.get(name, 2)


def _work_heads(case):
    t, heads, kh, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    values = t * (heads + kh) * d
    size = _size(case["dtype"])
    cached = t * kh * d * (size + 2 * min(size, 2)) + 8 * t if case["cached"] else 0
    return {"bytes": 2 * values * size + cached + 8 * t + 4 * case["rotary_dim"] + 8 * d,
            "flops": 8 * values}


def _work_cache(case):
    values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
    scales = 2 * 4 * 2 * case["tokens"] * case["kv_heads"] if case["held"] == "e4m3" else 0
    # the rows read and the held ones written, then the held ones read and the rows written
    return {"bytes": 2 * values * (_size(case["dtype"]) + _size(case["held"])) + scales
            + 16 * case["tokens"], "flops": 4 * values}


def _work_prompt(case):
    h, kh, d, before = case["heads"], case["kv_heads"], case["dim"], case["before"]
    lengths = _lengths(case)
    tokens, keys = sum(lengths), sum(n + before for n in lengths)
    pairs = sum(n * before + (n * (n + 1) // 2 if case["causal"] else n * n) for n in lengths)
    size = _size(case["dtype"])
    return {"bytes": size * d * (2 * tokens * h + 2 * keys * kh) + 8 * (len(lengths) + 1),
            "flops": 4 * pairs * h * d}


def _work_decode(case):
    b, h, kh, d, page = (case[n] for n in ("batch", "heads", "kv_heads", "dim", "page"))
    lengths = _lengths(case)
    rows = 2 * sum(lengths) * kh
    row = d * _size(case["held"]) + (4 if case["held"] == "e4m3" else 0)
    return {"bytes": rows * row + 2 * b * h * d * _size(case["dtype"]) + 4 * b
            + 4 * sum(-(-n // page) for n in lengths), "flops": 4 * sum(lengths) * h * d}
