"""Linear layers in 8-bit floating point (OCP E4M3, ``torch.float8_e4m3fn``) with a float32 scale
for each block of 128: weights per 128 x 128 block, activations per row and group of 128, as block
quantized checkpoints store them (``weight`` with ``weight_scale_inv`` [out / 128, in / 128];
sglang_omni/quantization.py:137-187 passes them through). The products run on the 8-bit matrix
cores; scales and sums are float32."""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from .. import _native as N

BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)


@dataclass
class BlockFp8Weight:
    """A linear layer's weight: E4M3 [out, in] (in a multiple of 16), one float32 scale per block of
    128 x 128 [ceil(out / 128), ceil(in / 128)], and an optional float32 bias [out]."""

    weight: torch.Tensor
    scale: torch.Tensor
    bias: torch.Tensor | None = None

    def to(self, device) -> "BlockFp8Weight":
        return BlockFp8Weight(self.weight.to(device), self.scale.to(device),
                              None if self.bias is None else self.bias.to(device))


@dataclass
class BlockFp8Rows:
    """Activation rows: E4M3 values [rows, features] and one float32 scale per row and group of 128
    features [rows, ceil(features / 128)], of any strides."""

    values: torch.Tensor
    scale: torch.Tensor

    def dequantized(self) -> torch.Tensor:
        """The float32 values the rows stand for."""
        full = self.scale.repeat_interleave(BLOCK, 1)[:, :self.values.shape[1]]
        return self.values.float() * full


def pack_block_fp8(weight: torch.Tensor, bias: torch.Tensor | None = None) -> BlockFp8Weight:
    """weight [out, in] (any float dtype) -> E4M3 with a scale per block of 128 x 128, scale =
    max|block| / 448 (1 for a block of zeros). Inputs short of a multiple of 16 are filled up with
    zero weights, as ``quantize_block_rows`` fills its rows."""
    if weight.dim() != 2:
        raise ValueError("a linear weight is [out_features, in_features]")
    n, k = weight.shape
    rb, cb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(rb * BLOCK, cb * BLOCK, dtype=torch.float32, device=weight.device)
    w[:n, :k] = weight.detach().float()
    w = w.view(rb, BLOCK, cb, BLOCK)
    amax = w.abs().amax((1, 3), keepdim=True)
    scale = torch.where(amax >= 2.0 ** -100, amax / 448.0, torch.ones_like(amax))
    q = (w / scale).to(_E4M3).view(rb * BLOCK, cb * BLOCK)[:n, :-(-k // 16) * 16]
    return BlockFp8Weight(q.contiguous(), scale.view(rb, cb).contiguous(),
                          None if bias is None else bias.detach().float().contiguous())


def block_fp8_weight(name: str, weight: torch.Tensor, scale_inv: torch.Tensor,
                     bias: torch.Tensor | None = None, *, inverted: bool = False) -> BlockFp8Weight:
    """A checkpoint's E4M3 linear weight and its ``weight_scale_inv`` [ceil(out / 128),
    ceil(in / 128)], checked as ``quantization.checkpoint_fp8_multiplier`` checks them;
    ``inverted`` checkpoints store the multiplier's reciprocal."""
    from ..quantization import checkpoint_fp8_multiplier

    if weight.dtype != _E4M3 or weight.dim() != 2 or weight.shape[1] % 16:
        raise ValueError(f"{name}: expected a float8_e4m3fn weight [out, in], in a multiple of 16")
    scale = checkpoint_fp8_multiplier(name, scale_inv, inverted=inverted)
    blocks = tuple(-(-d // BLOCK) for d in weight.shape)
    if tuple(scale.shape) != blocks:
        raise ValueError(f"{name}: block scales of shape {tuple(scale.shape)}, expected {blocks}")
    return BlockFp8Weight(weight.contiguous(), scale.contiguous(),
                          None if bias is None else bias.detach().float().contiguous())


def quantize_block_rows(x: torch.Tensor) -> BlockFp8Rows:
    """x [rows, features] (bf16, f16 or f32, contiguous rows) as E4M3 rows: each group of 128 takes
    scale = amax / 448 and q = E4M3(x * (448 / amax)). Rows are filled up with zeros to a multiple
    of 16 features."""
    N.require_device(x)
    if x.dim() != 2 or x.dtype not in _FLOATS or (x.stride(1) != 1 and x.shape[1] != 1):
        raise ValueError("x must be bf16, f16 or f32 [rows, features] with contiguous rows")
    rows, k = x.shape
    if k < 1:
        raise ValueError("x has no features")
    values = torch.empty(rows, (k + 15) // 16 * 16, dtype=_E4M3, device=x.device)
    scale = torch.empty(rows, (k + BLOCK - 1) // BLOCK, dtype=torch.float32, device=x.device)
    lib = N.load_library()
    N.check(lib.omni_block_quantize(x.data_ptr(), N.omni_dtype(x.dtype), N.row_stride(x), rows, k,
                                    values.data_ptr(), values.shape[1], scale.data_ptr(),
                                    scale.shape[1], N.stream_handle(x.device)),
            "omni_block_quantize")
    return BlockFp8Rows(values, scale)


def block_fp8_linear(x: torch.Tensor | BlockFp8Rows, weight: BlockFp8Weight,
                     out: torch.Tensor | None = None, *,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out = x @ W^T + bias [rows, out_features] on the current stream, float32 sums rounded once to
    out_dtype (bf16, f16 or f32; ``out``'s own when it is given). x is ``BlockFp8Rows``, or a float
    tensor [rows, in_features] that is quantized as ``quantize_block_rows`` does."""
    if not isinstance(x, BlockFp8Rows):
        x = quantize_block_rows(x)
    values, scale, w, ws = x.values, x.scale, weight.weight, weight.scale
    device = values.device
    N.require_device(values, scale, w, ws, weight.bias, out)
    if values.dtype != _E4M3 or w.dtype != _E4M3 or values.dim() != 2 or w.dim() != 2:
        raise ValueError("x and the weight must be float8_e4m3fn matrices")
    rows, k = values.shape
    n = w.shape[0]
    if w.shape[1] != k:
        raise ValueError(f"x has {k} features, the weight takes {w.shape[1]}")
    blocks = (k + BLOCK - 1) // BLOCK
    if (scale.dtype != torch.float32 or scale.shape != (rows, blocks)
            or ws.dtype != torch.float32 or ws.shape != ((n + BLOCK - 1) // BLOCK, blocks)
            or (ws.stride(1) != 1 and blocks > 1)):
        raise ValueError("scales must be float32 [rows, ceil(in / 128)] and "
                         "[ceil(out / 128), ceil(in / 128)]")
    if (values.stride(1) != 1 and k > 1) or (w.stride(1) != 1 and k > 1):
        raise ValueError("x and the weight must have contiguous rows")
    bias = weight.bias
    if bias is not None:
        N.require_vector(bias, n, "bias", device)
    if out is None:
        out = torch.empty(rows, n, dtype=out_dtype, device=device)
    elif out.shape != (rows, n) or (out.stride(1) != 1 and n > 1):
        raise ValueError(f"out must be [{rows}, {n}] with contiguous rows")
    if out.dtype not in _FLOATS:
        raise ValueError("out must be bf16, f16 or f32")
    if not (device == scale.device == w.device == ws.device == out.device):
        raise ValueError("x, the weight and out must be on one GPU")
    args = N.BlockFp8Args(values.data_ptr(), N.row_stride(values), scale.data_ptr(),
                          scale.stride(0), scale.stride(1), w.data_ptr(), N.row_stride(w),
                          ws.data_ptr(), N.row_stride(ws), rows, n, k, N.ptr(bias),
                          out.data_ptr(), N.row_stride(out), N.omni_dtype(out.dtype))
    lib = N.load_library()
    N.check(lib.omni_block_fp8_gemm(ctypes.byref(args), N.stream_handle(device)),
            "omni_block_fp8_gemm")
    return out


__all__ = ["BlockFp8Rows", "BlockFp8Weight", "block_fp8_linear", "block_fp8_weight",
           "pack_block_fp8", "quantize_block_rows"]
