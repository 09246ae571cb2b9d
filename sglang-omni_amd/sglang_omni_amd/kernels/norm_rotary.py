"""The query and key heads of a layer between its qkv product and its attention: an RMS norm over each
head and the rotary positions in one pass, and in the same launch the keys and values into the paged
cache."""

from __future__ import annotations

import torch

from .. import _native as N
from .kv_cache import PagedKvCache, _rows, _slots
from .rotary import _FLOATS, _LAYOUTS, _heads

_CODES, _pack = N.TORCH_TO_OMNI, N.pack_norm_rotary
_launch = None  # the entry point, bound at the first call


def _weight(weight: torch.Tensor | None, name: str, dim: int, index: int) -> int:
    if weight is None:
        return 0
    if weight.dtype is not torch.float32 or weight.dim() != 1 or weight.shape[0] != dim \
            or not weight.is_contiguous() or weight.get_device() != index:
        raise ValueError(f"{name} must be contiguous float32 [{dim}] on q's GPU")
    return weight.data_ptr()


def norm_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                inv_freq: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                k_weight: torch.Tensor | None = None, eps: float = 1e-6, layout: str = "half",
                factor: float = 1.0, v: torch.Tensor | None = None,
                cache: PagedKvCache | None = None, slots: torch.Tensor | None = None,
                q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None
                ) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """q [tokens, heads, dim] and k [tokens, kv_heads, dim] (or None), each head normed, x / sqrt(mean(x^2)
    + eps) * weight (float32 [dim], optional), then turned at positions [tokens] as ``apply_rotary`` does
    (inv_freq, layout and factor as there), float32 throughout and rounded once; on the current stream.
    Returns the outputs (q's alone without k).

    With ``cache``, ``v`` [tokens, kv_heads, dim] and ``slots`` [tokens], k's outputs and v also go into
    the cache as ``write_kv_cache`` puts them there, in the same launch and with the same bits.

    bf16, f16 or f32, dim up to 512; views of a qkv buffer are taken as they are; q_out / k_out may be q /
    k themselves."""
    index = q.get_device()
    if index < 0 or positions.get_device() != index or inv_freq.get_device() != index \
            or (k is not None and k.get_device() != index):
        N.require_device(q, k, positions, inv_freq)
        raise ValueError("q, k, positions and inv_freq must be on one GPU")
    q_token, q_head = _heads(q, "q")
    shape, dtype = q.shape, q.dtype
    tokens, heads, dim = shape
    if dtype not in _FLOATS or heads < 1 or not 2 <= dim <= 512:
        raise ValueError("q must be bf16, f16 or f32, with at least one head of 2 to 512 values")
    if layout not in _LAYOUTS:
        raise ValueError(f"unknown layout {layout!r}")
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64 [pairs]")
    pairs = inv_freq.shape[0]
    if pairs < 1 or 2 * pairs > dim:
        raise ValueError(f"{pairs} pairs do not fit heads of {dim}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    if positions.dim() != 1 or positions.shape[0] != tokens \
            or positions.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"positions must be int32 or int64 [{tokens}]")
    if q_out is None:
        q_out = torch.empty_like(q)
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
        if k_shape[0] != tokens or kv_heads < 1 or k_shape[2] != dim or k.dtype is not dtype:
            raise ValueError("k must be [tokens, kv_heads, dim] of q's dtype, with at least one head")
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
    v_ptr = v_token = v_head = address = 0
    slot_args = (0, 0, 0)
    if cache is not None:
        if k is None or v is None or slots is None:
            raise ValueError("a cache takes k, v and slots")
        if cache.index != index or v.get_device() != index:
            raise ValueError("q, v and the cache must be on one GPU")
        _rows(k, "k", cache)
        v_token, v_head = _rows(v, "v", cache)
        if v.shape[0] != tokens or v.dtype is not dtype:
            raise ValueError("v must be like k")
        v_ptr, address, slot_args = v.data_ptr(), cache.address, _slots(slots, tokens, index)
    elif v is not None or slots is not None:
        raise ValueError("v and slots go with a cache")
    args = _pack(
        q.data_ptr(), q_token, q_head, k_ptr, k_token, k_head, v_ptr, v_token, v_head,
        q_out.data_ptr(), qo_token, qo_head, ko_ptr, ko_token, ko_head, _CODES[dtype], tokens, heads,
        kv_heads, dim, 1, _weight(q_weight, "q_weight", dim, index),
        _weight(k_weight, "k_weight", dim, index), eps, pairs, positions.data_ptr(),
        _CODES[positions.dtype], positions.stride(0), inv_freq.data_ptr(), factor, _LAYOUTS[layout],
        address, *slot_args)
    global _launch
    if _launch is None:
        _launch = N.load_library().omni_norm_rotary
    status = N.launch_on(index, _launch, args)
    if status:
        N.check(status, "omni_norm_rotary")
    return q_out if k is None else (q_out, k_out)


__all__ = ["norm_rotary"]
