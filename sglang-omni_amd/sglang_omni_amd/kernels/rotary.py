"""Rotary positions: half and interleaved pair layouts, the whole head or its first part, and
frequencies scaled for long contexts. Angles are formed in float64 from the positions and float64
frequencies, so they stay exact at any position a context reaches."""

from __future__ import annotations

import ctypes
import math
from typing import Any, Mapping

import torch

from .. import _native as N

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_LAYOUTS = {"half": N.ROTARY_HALF, "interleaved": N.ROTARY_INTERLEAVED}


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
      pair index; the factor is "attention_factor" or 0.1 ln(factor) + 1
    - "longrope": divided by "long_factor" (or "short_factor" with "short": True), one per pair; the
      factor is "attention_factor" or sqrt(1 + ln(factor) / ln(original context))
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not base > 1.0:
        raise ValueError(f"base must be above 1, got {base}")
    pairs = rotary_dim // 2
    inv = float(base) ** (-torch.arange(pairs, dtype=torch.float64) * 2 / rotary_dim)
    scaling = dict(scaling or {})
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    factor = float(scaling.get("factor", 1.0))
    if not factor >= 1.0:
        raise ValueError(f"the scaling factor must be at least 1, got {factor}")
    cos_factor = 1.0
    if kind == "linear":
        inv = inv / factor
    elif kind == "llama3":
        original = float(scaling["original_max_position_embeddings"])
        low, high = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not high > low:
            raise ValueError("high_freq_factor must be above low_freq_factor")
        turns = original * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / factor)
    elif kind == "yarn":
        original = float(scaling["original_max_position_embeddings"])

        def pair(turns: float) -> float:
            return rotary_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = max(math.floor(pair(float(scaling.get("beta_fast", 32)))), 0)
        high = min(math.ceil(pair(float(scaling.get("beta_slow", 1)))), rotary_dim - 1)
        ramp = (torch.arange(pairs, dtype=torch.float64) - low) / max(high - low, 1e-3)
        ramp = ramp.clamp(0, 1)
        inv = inv * (1 - ramp) + inv / factor * ramp
        cos_factor = float(scaling.get("attention_factor") or 0.1 * math.log(factor) + 1.0)
    elif kind == "longrope":
        name = "short_factor" if scaling.get("short") else "long_factor"
        per_pair = torch.as_tensor(scaling[name], dtype=torch.float64)
        if per_pair.shape != (pairs,):
            raise ValueError(f"{name} must hold {pairs} values")
        inv = inv / per_pair
        original = float(scaling["original_max_position_embeddings"])
        cos_factor = float(scaling.get("attention_factor")
                           or math.sqrt(1 + math.log(factor) / math.log(original)))
    elif kind != "default":
        raise ValueError(f"unknown rope scaling {kind!r}")
    return inv.to(device) if device is not None else inv, cos_factor


def _check_heads(t: torch.Tensor, name: str) -> None:
    if t.dim() != 3 or (t.stride(2) != 1 and t.shape[2] > 1):
        raise ValueError(f"{name} must be [tokens, heads, dim] with contiguous dim")


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
    N.require_device(q, k, positions, inv_freq, q_out, k_out)
    _check_heads(q, "q")
    tokens, heads, dim = q.shape
    device, dtype = q.device, q.dtype
    if dtype not in _FLOATS:
        raise ValueError("q must be bf16, f16 or f32")
    if layout not in _LAYOUTS:
        raise ValueError(f"unknown layout {layout!r}")
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64 [pairs]")
    pairs = inv_freq.shape[0]
    if pairs < 1 or 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs do not fit heads of {dim}")
    if positions.shape != (tokens,) or positions.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"positions must be int32 or int64 [{tokens}]")
    if positions.device != device or inv_freq.device != device:
        raise ValueError("q, positions and inv_freq must be on one GPU")
    if heads < 1:
        raise ValueError("q has no heads")
    if q_out is None:
        q_out = torch.empty(tokens, heads, dim, dtype=dtype, device=device)
    else:
        _check_heads(q_out, "q_out")
        if q_out.shape != q.shape or q_out.dtype != dtype or q_out.device != device:
            raise ValueError("q_out must be like q")
    kv_heads, k_ptr, k_t, k_h, ko_ptr, ko_t, ko_h = 0, None, 0, 0, None, 0, 0
    if k is not None:
        _check_heads(k, "k")
        kv_heads = k.shape[1]
        if k.shape[0] != tokens or k.shape[2] != dim or k.dtype != dtype or k.device != device:
            raise ValueError("k must be [tokens, kv_heads, dim] of q's dtype and device")
        if k_out is None:
            k_out = torch.empty(tokens, kv_heads, dim, dtype=dtype, device=device)
        else:
            _check_heads(k_out, "k_out")
            if k_out.shape != k.shape or k_out.dtype != dtype or k_out.device != device:
                raise ValueError("k_out must be like k")
        k_ptr, k_t, k_h = k.data_ptr(), k.stride(0), k.stride(1)
        ko_ptr, ko_t, ko_h = k_out.data_ptr(), k_out.stride(0), k_out.stride(1)
    elif k_out is not None:
        raise ValueError("k_out goes with k")
    args = N.RotaryArgs(q.data_ptr(), q.stride(0), q.stride(1), k_ptr, k_t, k_h, q_out.data_ptr(),
                        q_out.stride(0), q_out.stride(1), ko_ptr, ko_t, ko_h, N.omni_dtype(dtype),
                        tokens, heads, kv_heads, dim, pairs, positions.data_ptr(),
                        N.omni_dtype(positions.dtype), positions.stride(0), inv_freq.data_ptr(),
                        factor, _LAYOUTS[layout], int(transposed))
    lib = N.load_library()
    N.check(lib.omni_rotary(ctypes.byref(args), N.stream_handle(device)), "omni_rotary")
    return q_out if k is None else (q_out, k_out)


__all__ = ["apply_rotary", "rotary_frequencies"]
