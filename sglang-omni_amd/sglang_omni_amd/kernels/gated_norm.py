"""The step between two blocks of a transformer in one launch: the norm after a block, its gate and
residual scale, the residual add, and the norm before the next block, optionally straight to the
8-bit rows of the next block's linear layers."""

from __future__ import annotations

import ctypes

import torch

from .. import _native as N
from .block_fp8 import BLOCK, BlockFp8Rows

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_NORMS = {"rms": N.NORM_RMS, "layer": N.NORM_LAYER}
_ACTIVATIONS = {"none": N.GATE_NONE, "sigmoid": N.GATE_SIGMOID, "tanh": N.GATE_TANH}


def gated_residual_norm(x: torch.Tensor, y: torch.Tensor, *, norm: str = "rms", eps: float = 1e-6,
                        post_norm: bool = False, post_weight: torch.Tensor | None = None,
                        post_bias: torch.Tensor | None = None,
                        pre_weight: torch.Tensor | None = None,
                        pre_bias: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                        gate_activation: str = "none", scale: float = 1.0,
                        normed_dtype: torch.dtype | None = None,
                        residual_out: torch.Tensor | None = None
                        ) -> tuple[torch.Tensor, torch.Tensor | BlockFp8Rows]:
    """(residual, normed) on the current stream:

        u = post_norm(y) * post_weight + post_bias     (y itself without post_norm)
        h = x + scale * act(gate) * u                  residual: h rounded to x's dtype
        normed = norm(h) * pre_weight + pre_bias       from h before that rounding

    x, y [rows, channels] with contiguous rows, y bf16 / f16 / f32, x of y's dtype or float32.
    ``norm`` is "rms" or "layer" (biases with "layer" only); weights and biases float32 [channels].
    gate is [channels], or [G, channels] with rows % G == 0: rows / G consecutive rows share a gate
    (one per sequence; one per token with G = rows). normed has ``normed_dtype`` (y's by default);
    with ``torch.float8_e4m3fn`` it is ``BlockFp8Rows``. ``residual_out`` may be x."""
    N.require_device(x, y, gate, residual_out)
    if x.dim() != 2 or x.shape != y.shape or x.stride(1) != 1 and x.shape[1] > 1 \
            or y.stride(1) != 1 and y.shape[1] > 1:
        raise ValueError("x and y must be [rows, channels] alike, with contiguous rows")
    if y.dtype not in _FLOATS or (x.dtype != y.dtype and x.dtype != torch.float32):
        raise ValueError("y must be bf16, f16 or f32, and x of y's dtype or float32")
    if norm not in _NORMS or gate_activation not in _ACTIVATIONS:
        raise ValueError(f"unknown norm {norm!r} or gate activation {gate_activation!r}")
    rows, c = x.shape
    device = x.device
    if c < 1:
        raise ValueError("x has no channels")
    if norm == "rms" and (post_bias is not None or pre_bias is not None):
        raise ValueError("biases go with the layer norm")
    if not post_norm and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias go with post_norm")
    if post_weight is not None:
        N.require_vector(post_weight, c, "post_weight", device)
    if post_bias is not None:
        N.require_vector(post_bias, c, "post_bias", device)
    if pre_weight is not None:
        N.require_vector(pre_weight, c, "pre_weight", device)
    if pre_bias is not None:
        N.require_vector(pre_bias, c, "pre_bias", device)
    if y.device != device or (gate is not None and gate.device != device):
        raise ValueError("x, y and gate must be on one GPU")
    gate_ptr, gate_dtype, gate_stride, rows_per_gate = None, N.DTYPE_F32, 0, 1
    if gate is not None:
        gates = 1 if gate.dim() == 1 else gate.shape[0]
        if (gate.dim() not in (1, 2) or gate.shape[-1] != c or gate.dtype not in _FLOATS
                or (gate.stride(-1) != 1 and c > 1) or gates < 1 or rows % gates):
            raise ValueError("gate must be bf16, f16 or f32 [channels] or [G, channels], rows a "
                             "multiple of G, with contiguous rows")
        gate_ptr, gate_dtype = gate.data_ptr(), N.omni_dtype(gate.dtype)
        # a stride of 0 is a gate expanded over its rows
        gate_stride = gate.stride(0) if gate.dim() == 2 else 0
        rows_per_gate = max(rows // gates, 1)
    elif gate_activation != "none":
        raise ValueError("gate_activation goes with a gate")
    if residual_out is None:
        residual_out = torch.empty(rows, c, dtype=x.dtype, device=device)
    elif (residual_out.shape != x.shape or residual_out.dtype != x.dtype
          or (residual_out.stride(1) != 1 and c > 1) or residual_out.device != device):
        raise ValueError("residual_out must be like x, with contiguous rows")
    dtype = y.dtype if normed_dtype is None else normed_dtype
    normed_scale = None
    if dtype == torch.float8_e4m3fn:
        normed = torch.empty(rows, (c + 15) // 16 * 16, dtype=dtype, device=device)
        normed_scale = torch.empty(rows, (c + BLOCK - 1) // BLOCK, dtype=torch.float32,
                                   device=device)
    elif dtype in _FLOATS:
        normed = torch.empty(rows, c, dtype=dtype, device=device)
    else:
        raise ValueError("normed_dtype must be bf16, f16, f32 or float8_e4m3fn")
    args = N.GatedNormArgs(
        x.data_ptr(), N.omni_dtype(x.dtype), N.row_stride(x), y.data_ptr(),
        N.omni_dtype(y.dtype), N.row_stride(y), rows, c, _NORMS[norm],
        int(post_norm), eps, scale, N.ptr(post_weight), N.ptr(post_bias), N.ptr(pre_weight),
        N.ptr(pre_bias), gate_ptr, gate_dtype, gate_stride, rows_per_gate,
        _ACTIVATIONS[gate_activation], residual_out.data_ptr(),
        N.row_stride(residual_out), normed.data_ptr(), N.omni_dtype(dtype),
        normed.shape[1], N.ptr(normed_scale), 0 if normed_scale is None else normed_scale.shape[1])
    lib = N.load_library()
    N.check(lib.omni_gated_residual_norm(ctypes.byref(args), N.stream_handle(device)),
            "omni_gated_residual_norm")
    return residual_out, normed if normed_scale is None else BlockFp8Rows(normed, normed_scale)


__all__ = ["gated_residual_norm"]
