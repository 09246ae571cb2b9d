"""The step between two blocks of a transformer in one launch: the norm after a block, its gate and
residual scale, the residual add, and the norm before the next block, optionally straight to the
8-bit rows of the next block's linear layers."""

from __future__ import annotations

import torch

from .. import _native as N
from .block_fp8 import BLOCK, BlockFp8Rows

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CODES, _pack, _raw_stream = N.TORCH_TO_OMNI, N.pack_gated_norm, N.raw_stream
_launch = None  # the entry point, bound at the first call
_NORMS = {"rms": N.NORM_RMS, "layer": N.NORM_LAYER}
_ACTIVATIONS = {"none": N.GATE_NONE, "sigmoid": N.GATE_SIGMOID, "tanh": N.GATE_TANH}


def _vector(t: torch.Tensor | None, channels: int, index: int, what: str) -> int:
    """The address of a per-channel float32 vector on GPU ``index``, 0 for none."""
    if t is None:
        return 0
    if t.dtype is not torch.float32 or t.numel() != channels or t.get_device() != index \
            or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous float32 [{channels}] on x's GPU")
    return t.data_ptr()


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
    index = x.get_device()
    if index < 0 or y.get_device() != index or (gate is not None and gate.get_device() != index):
        N.require_device(x, y, gate)
        raise ValueError("x, y and gate must be on one GPU")
    x_dtype, y_dtype = x.dtype, y.dtype
    shape = x.shape
    if len(shape) != 2 or shape != y.shape:
        raise ValueError("x and y must be [rows, channels] alike")
    rows, c = shape
    x_stride, x_contiguous = x.stride()
    y_stride, y_contiguous = y.stride()
    if c < 1 or (c > 1 and (x_contiguous != 1 or y_contiguous != 1)):
        raise ValueError("x and y must have contiguous rows of at least one channel")
    if y_dtype not in _FLOATS or (x_dtype is not y_dtype and x_dtype is not torch.float32):
        raise ValueError("y must be bf16, f16 or f32, and x of y's dtype or float32")
    if norm not in _NORMS or gate_activation not in _ACTIVATIONS:
        raise ValueError(f"unknown norm {norm!r} or gate activation {gate_activation!r}")
    if norm == "rms" and (post_bias is not None or pre_bias is not None):
        raise ValueError("biases go with the layer norm")
    if not post_norm and (post_weight is not None or post_bias is not None):
        raise ValueError("post_weight and post_bias go with post_norm")
    gate_ptr, gate_code, gate_stride, rows_per_gate = 0, N.DTYPE_F32, 0, 1
    if gate is not None:
        gate_shape, gate_strides = gate.shape, gate.stride()
        gates = gate_shape[0] if len(gate_shape) == 2 else 1
        if (len(gate_shape) not in (1, 2) or gate_shape[-1] != c or gate.dtype not in _FLOATS
                or (c > 1 and gate_strides[-1] != 1) or gates < 1 or rows % gates):
            raise ValueError("gate must be bf16, f16 or f32 [channels] or [G, channels], rows a "
                             "multiple of G, with contiguous rows")
        gate_ptr, gate_code = gate.data_ptr(), _CODES[gate.dtype]
        if gates > 1:
            gate_stride = gate_strides[0]  # 0 for a gate expanded over its rows
        rows_per_gate = max(rows // gates, 1)
    elif gate_activation != "none":
        raise ValueError("gate_activation goes with a gate")
    if residual_out is None:
        residual_out = torch.empty_like(x)
        out_stride = residual_out.stride(0) if rows > 1 else c
    else:
        if (residual_out.shape != shape or residual_out.dtype is not x_dtype
                or (c > 1 and residual_out.stride(1) != 1) or residual_out.get_device() != index):
            raise ValueError("residual_out must be like x, with contiguous rows")
        out_stride = N.row_stride(residual_out)
    if normed_dtype is None:
        normed_dtype = y_dtype
    normed_scale, scale_ptr, scale_stride = None, 0, 0
    if normed_dtype is y_dtype:
        normed = torch.empty_like(y)
    elif normed_dtype in _FLOATS:
        normed = torch.empty(shape, dtype=normed_dtype, device=x.device)
    elif normed_dtype is torch.float8_e4m3fn:
        normed = torch.empty((rows, (c + 15) // 16 * 16), dtype=normed_dtype, device=x.device)
        scale_stride = (c + BLOCK - 1) // BLOCK
        normed_scale = torch.empty((rows, scale_stride), dtype=torch.float32, device=x.device)
        scale_ptr = normed_scale.data_ptr()
    else:
        raise ValueError("normed_dtype must be bf16, f16, f32 or float8_e4m3fn")
    args = _pack(
        x.data_ptr(), _CODES[x_dtype], x_stride if rows > 1 else c, y.data_ptr(), _CODES[y_dtype],
        y_stride if rows > 1 else c, rows, c, _NORMS[norm], 1 if post_norm else 0, eps, scale,
        _vector(post_weight, c, index, "post_weight"), _vector(post_bias, c, index, "post_bias"),
        _vector(pre_weight, c, index, "pre_weight"), _vector(pre_bias, c, index, "pre_bias"),
        gate_ptr, gate_code, gate_stride, rows_per_gate, _ACTIVATIONS[gate_activation],
        residual_out.data_ptr(), out_stride, normed.data_ptr(), _CODES[normed_dtype],
        N.row_stride(normed), scale_ptr, scale_stride)
    global _launch
    if _launch is None:
        _launch = N.load_library().omni_gated_residual_norm
    status = _launch(args, _raw_stream(index))
    if status:
        N.check(status, "omni_gated_residual_norm")
    return residual_out, normed if normed_scale is None else BlockFp8Rows(normed, normed_scale)


__all__ = ["gated_residual_norm"]
