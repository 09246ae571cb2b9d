"""Rotary positions: half and interleaved pair layouts, the whole head or its first part, and
frequencies scaled for long contexts. Angles are formed in float64 from the positions and float64
frequencies, so they stay exact at any position a context reaches."""

from __future__ import annotations

import math
from typing import Any, Mapping

import torch

from .. import _native as N

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CODES, _pack, _raw_stream = N.TORCH_TO_OMNI, N.pack_rotary, N.raw_stream
_launch = None  # the entry point, bound at the first call
_LAYOUTS = {"half": N.ROTARY_HALF, "interleaved": N.ROTARY_INTERLEAVED}


# The keys of each kind of scaling. Another key would change what the configuration means, so it is
# refused rather than passed over.
_SCALING_KEYS = {
    "default": set(),
    "linear": {"factor"},
    "llama3": {"factor", "original_max_position_embeddings", "low_freq_factor", "high_freq_factor"},
    "yarn": {"factor", "original_max_position_embeddings", "beta_fast", "beta_slow",
             "attention_factor", "mscale", "mscale_all_dim", "truncate"},
    "longrope": {"factor", "original_max_position_embeddings", "attention_factor", "long_factor",
                 "short_factor", "short"},
}


def _yarn_magnitude(factor: float, mscale: float) -> float:
    return 0.1 * mscale * math.log(factor) + 1.0


def rotary_frequencies(rotary_dim: int, base: float = 10000.0,
                       scaling: Mapping[str, Any] | None = None,
                       device: torch.device | str | None = None) -> tuple[torch.Tensor, float]:
    """(radians per position of each pair, float64 [rotary_dim / 2]; the factor on cos and sin) for
    ``apply_rotary``. ``scaling`` is a configuration's rope scaling, by its "rope_type" (or "type"):

    - "default": base ** (-2 i / rotary_dim), factor 1
    - "linear": divided by "factor"
    - "llama3": pairs that turn less than "low_freq_factor" times in
      "original_max_position_embeddings" divided by "factor", those that turn more than
      "high_freq_factor" times kept, between them a blend by the turns
    - "yarn": pairs that turn less than "beta_slow" (1) times in the original context divided by
      "factor", those that turn more than "beta_fast" (32) times kept, between them a ramp over the
      pair index, its ends rounded outwards to whole pairs unless "truncate" is False; the factor is
      "attention_factor", or m("mscale") / m("mscale_all_dim") where both are given, m(s) = 0.1 s
      ln(factor) + 1, or else m(1)
    - "longrope": divided by "long_factor" (or "short_factor" with "short": True), one per pair; the
      factor is "attention_factor" or sqrt(1 + ln(factor) / ln(original context)), where "factor" is
      the ratio of the model's context to the original one

    A null value is an absent one. "rope_theta" must be ``base``; any other key, a missing "factor"
    or a missing context (but longrope's with an "attention_factor") is a ValueError: sections of
    several position rows and a partial head, for instance, are the caller's to apply."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not base > 1.0:
        raise ValueError(f"base must be above 1, got {base}")
    pairs = rotary_dim // 2
    inv = float(base) ** (-torch.arange(pairs, dtype=torch.float64) * 2 / rotary_dim)
    scaling = {key: value for key, value in (scaling or {}).items() if value is not None}
    kinds = {scaling.pop(key) for key in ("rope_type", "type") if key in scaling} or {"default"}
    kind = kinds.pop()
    if kinds or kind not in _SCALING_KEYS:
        raise ValueError(f"unknown rope scaling {' / '.join(map(repr, (kind, *kinds)))}")
    if float(scaling.pop("rope_theta", base)) != float(base):
        raise ValueError(f"the rope scaling's rope_theta is not the base {base}")
    unknown = sorted(scaling.keys() - _SCALING_KEYS[kind])
    if unknown:
        raise ValueError(f"{kind} rope scaling does not take {', '.join(unknown)}")

    def number(key: str) -> float:
        if key not in scaling:
            raise ValueError(f"{kind} rope scaling needs {key}")
        return float(scaling[key])

    def context() -> float:
        original = number("original_max_position_embeddings")
        if not original > 1.0:
            raise ValueError(f"the original context must be above 1, got {original}")
        return original

    factor = 1.0
    if kind != "default" and not (kind == "longrope" and "attention_factor" in scaling):
        factor = number("factor")
        if not factor >= 1.0:
            raise ValueError(f"the scaling factor must be at least 1, got {factor}")
    cos_factor = 1.0
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        original = context()
        low, high = number("low_freq_factor"), number("high_freq_factor")
        if not high > low:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        turns = original * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / factor)
    elif kind == "yarn":
        original = context()

        def pair(turns: float) -> float:
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = pair(float(scaling.get("beta_fast", 32))), pair(float(scaling.get("beta_slow", 1)))
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, rotary_dim - 1)
        if low > high:  # beta_fast below beta_slow, or a context of less than a turn
            raise ValueError("yarn's ramp ends before it begins")
        ramp = (torch.arange(pairs, dtype=torch.float64) - low) / max(high - low, 1e-3)
        ramp = ramp.clamp(0, 1)
        inv = inv * (1 - ramp) + inv / factor * ramp
        mscale = float(scaling.get("mscale", 1.0))
        mscale_all_dim = float(scaling.get("mscale_all_dim", 0.0))
        if "attention_factor" in scaling:
            cos_factor = float(scaling["attention_factor"])
        elif mscale and mscale_all_dim and "mscale" in scaling:
            cos_factor = _yarn_magnitude(factor, mscale) / _yarn_magnitude(factor, mscale_all_dim)
        elif mscale == 1.0 and mscale_all_dim == 0.0:
            cos_factor = _yarn_magnitude(factor, 1.0)
        else:  # the published definitions differ on one without the other
            raise ValueError("yarn's mscale and mscale_all_dim come together")
    elif kind == "longrope":
        name = "short_factor" if scaling.get("short") else "long_factor"
        if name not in scaling:
            raise ValueError(f"longrope rope scaling needs {name}")
        per_pair = torch.as_tensor(scaling[name], dtype=torch.float64)
        if per_pair.shape != (pairs,):
            raise ValueError(f"{name} must hold {pairs} values")
        inv = inv / per_pair
        cos_factor = (float(scaling["attention_factor"]) if "attention_factor" in scaling
                      else math.sqrt(1 + math.log(factor) / math.log(context())))
    return inv.to(device) if device is not None else inv, cos_factor


def _heads(t: torch.Tensor, name: str) -> tuple[int, int]:
    """The token and head strides of [tokens, heads, dim] with contiguous dim."""
    strides = t.stride()
    if len(strides) != 3 or (strides[2] != 1 and t.shape[2] > 1):
        raise ValueError(f"{name} must be [tokens, heads, dim] with contiguous dim")
    return strides[0], strides[1]


def apply_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 inv_freq: torch.Tensor, *, layout: str = "half", factor: float = 1.0,
                 transposed: bool = False, q_out: torch.Tensor | None = None,
                 k_out: torch.Tensor | None = None
                 ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """q [tokens, heads, dim] and k [tokens, kv_heads, dim] (or None) turned at positions [tokens]
    (int32 / int64) on the current stream; returns the outputs (q's alone without k). The first
    2 * len(inv_freq) values of a head are turned, the rest copied: pair i becomes
    (a cos - b sin, b cos + a sin) * factor, angle = position * inv_freq[i], with pairs (i, i +
    len(inv_freq)) in the "half" layout and (2 i, 2 i + 1) "interleaved". ``transposed`` turns back
    (by the negative angle), which is the gradient. bf16, f16 or f32; views of a qkv buffer are
    taken as they are; q_out / k_out may be q / k themselves."""
    index = q.get_device()
    if index < 0 or positions.get_device() != index or inv_freq.get_device() != index \
            or (k is not None and k.get_device() != index):
        N.require_device(q, k, positions, inv_freq)
        raise ValueError("q, k, positions and inv_freq must be on one GPU")
    q_token, q_head = _heads(q, "q")
    shape, dtype = q.shape, q.dtype
    tokens, heads, dim = shape
    if dtype not in _FLOATS or heads < 1:
        raise ValueError("q must be bf16, f16 or f32, with at least one head")
    if layout not in _LAYOUTS:
        raise ValueError(f"unknown layout {layout!r}")
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64 [pairs]")
    pairs = inv_freq.shape[0]
    if pairs < 1 or 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs do not fit heads of {dim}")
    positions_dtype = positions.dtype
    if positions.dim() != 1 or positions.shape[0] != tokens or (positions_dtype is not torch.int64
                                        and positions_dtype is not torch.int32):
        raise ValueError(f"positions must be int32 or int64 [{tokens}]")
    if q_out is None:
        q_out = torch.empty_like(q)  # dense, in q's order of tokens and heads
        qo_token, qo_head, _ = q_out.stride()
    else:
        qo_token, qo_head = _heads(q_out, "q_out")
        if q_out.shape != shape or q_out.dtype is not dtype or q_out.get_device() != index:
            raise ValueError("q_out must be like q")
    kv_heads = k_ptr = k_token = k_head = ko_ptr = ko_token = ko_head = 0
    if k is not None:
        k_token, k_head = _heads(k, "k")
        k_shape = k.shape
        kv_heads = k_shape[1]
        if k_shape[0] != tokens or k_shape[2] != dim or k.dtype is not dtype:
            raise ValueError("k must be [tokens, kv_heads, dim] of q's dtype")
        if k_out is None:
            k_out = torch.empty_like(k)
            ko_token, ko_head, _ = k_out.stride()
        else:
            ko_token, ko_head = _heads(k_out, "k_out")
            if k_out.shape != k_shape or k_out.dtype is not dtype or k_out.get_device() != index:
                raise ValueError("k_out must be like k")
        k_ptr, ko_ptr = k.data_ptr(), k_out.data_ptr()
    elif k_out is not None:
        raise ValueError("k_out goes with k")
    args = _pack(
        q.data_ptr(), q_token, q_head, k_ptr, k_token, k_head, q_out.data_ptr(), qo_token, qo_head,
        ko_ptr, ko_token, ko_head, _CODES[dtype], tokens, heads, kv_heads, dim, pairs,
        positions.data_ptr(), _CODES[positions_dtype], positions.stride(0), inv_freq.data_ptr(),
        factor, _LAYOUTS[layout], 1 if transposed else 0)
    global _launch
    if _launch is None:
        _launch = N.load_library().omni_rotary
    status = _launch(args, _raw_stream(index))
    if status:
        N.check(status, "omni_rotary")
    return q_out if k is None else (q_out, k_out)


__all__ = ["apply_rotary", "rotary_frequencies"]
