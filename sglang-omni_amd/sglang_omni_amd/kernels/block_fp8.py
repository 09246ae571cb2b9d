"""Linear layers in 8-bit floating point (OCP E4M3, ``torch.float8_e4m3fn``) with a float32 scale
for each block of 128: weights per 128 x 128 block, activations per row and group of 128, as block
quantized checkpoints store them (``weight`` with ``weight_scale_inv`` [out / 128, in / 128];
sglang_omni/quantization.py:137-187 passes them through). The products run on the 8-bit matrix
cores; scales and sums are float32."""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _native as N

BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CODES, _pack, _raw_stream = N.TORCH_TO_OMNI, N.pack_block_fp8, N.raw_stream
_launch = None  # the entry point, bound at the first call


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
    max|block| / 448 (1 for a block of zeros). NaN stays NaN and leaves the scale to the others; an
    infinity makes it infinite, so that every product with the block is NaN. Inputs short of a
    multiple of 16 are filled up with zero weights, as ``quantize_block_rows`` fills its rows."""
    if weight.dim() != 2:
        raise ValueError("a linear weight is [out_features, in_features]")
    n, k = weight.shape
    rb, cb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.zeros(rb * BLOCK, cb * BLOCK, dtype=torch.float32, device=weight.device)
    w[:n, :k] = weight.detach().float()
    w = w.view(rb, BLOCK, cb, BLOCK)
    amax = w.abs().nan_to_num(0.0, posinf=float("inf")).amax((1, 3), keepdim=True)
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
    """out = x @ W^T + bias [rows, out_features] on the current stream, summed in float32 and rounded
    once to out_dtype (bf16, f16 or f32; ``out``'s own when it is given). x is ``BlockFp8Rows``, or a float
    tensor [rows, features] that is quantized as ``quantize_block_rows`` does, to the same bits. A
    row's bits do not depend on the rows beside it.

    bf16 outputs multiply on the 8-bit matrix cores, which lose up to 7 * 2^-13 of the largest product
    of each 8 features (far less than the bf16 rounding, unless larger products cancel); f16 and f32
    ones on the bf16 matrix cores, exact products in float32 sums, at about half the rate: a bf16
    result of float32 sums is ``out_dtype=torch.float32`` and a cast."""
    w, w_scale, bias = weight.weight, weight.scale, weight.bias
    if type(x) is BlockFp8Rows:
        values, scale = x.values, x.scale
    else:
        values, scale = x, None
    index = values.get_device()
    if index < 0 or w.get_device() != index or w_scale.get_device() != index \
            or (scale is not None and scale.get_device() != index) \
            or (out is not None and out.get_device() != index):
        N.require_device(values, scale, w, w_scale, out)
        raise ValueError("x, the weight and out must be on one GPU")
    if w.dtype is not _E4M3 or w.dim() != 2 or values.dim() != 2:
        raise ValueError("the weight must be a float8_e4m3fn matrix, x a matrix")
    rows, features = values.shape
    n, k = w.shape
    blocks = (k + BLOCK - 1) // BLOCK
    x_stride, x_contiguous = values.stride()
    w_stride, w_contiguous = w.stride()
    if (x_contiguous != 1 and features > 1) or (w_contiguous != 1 and k > 1):
        raise ValueError("x and the weight must have contiguous rows")
    if w_scale.dtype is not torch.float32 or w_scale.shape != ((n + BLOCK - 1) // BLOCK, blocks) \
            or (blocks > 1 and w_scale.stride(1) != 1):
        raise ValueError("the weight's scale must be float32 [ceil(out / 128), ceil(in / 128)] with "
                         "contiguous rows")
    workspace, workspace_bytes = None, 0
    if scale is not None:
        if values.dtype is not _E4M3 or features != k:
            raise ValueError(f"x must be float8_e4m3fn rows of the weight's {k} features")
        if scale.dtype is not torch.float32 or scale.shape != (rows, blocks):
            raise ValueError("x's scale must be float32 [rows, ceil(in / 128)]")
        scale_ptr = scale.data_ptr()
        scale_row, scale_block = scale.stride()
    else:
        if values.dtype not in _FLOATS:
            raise ValueError("x must be BlockFp8Rows, or bf16, f16 or f32 rows")
        if (features + 15) // 16 * 16 != k:
            raise ValueError(f"x has {features} features, the weight takes {k}")
        scale_ptr = scale_row = scale_block = 0
        if rows > N.BLOCK_FP8_FEW_ROWS:
            workspace_bytes = rows * (k + 4 * blocks)
            workspace = torch.empty(workspace_bytes, dtype=torch.uint8, device=values.device)
    if bias is not None:
        N.require_vector(bias, n, "bias", values.device)
    if out is None:
        if out_dtype not in _FLOATS:
            raise ValueError("out must be bf16, f16 or f32")
        out = torch.empty((rows, n), dtype=out_dtype, device=values.device)
        out_stride = n
    else:
        out_dtype = out.dtype
        if out.shape != (rows, n) or (n > 1 and out.stride(1) != 1) or out_dtype not in _FLOATS:
            raise ValueError(f"out must be bf16, f16 or f32 [{rows}, {n}] with contiguous rows")
        out_stride = N.row_stride(out)
    args = _pack(
        values.data_ptr(), _CODES[values.dtype], x_stride if rows > 1 else features, features,
        scale_ptr, scale_row, scale_block, w.data_ptr(), w_stride if n > 1 else k,
        w_scale.data_ptr(), N.row_stride(w_scale), rows, n, k,
        0 if bias is None else bias.data_ptr(), out.data_ptr(), out_stride, _CODES[out_dtype],
        0 if workspace is None else workspace.data_ptr(), workspace_bytes)
    global _launch
    if _launch is None:
        _launch = N.load_library().omni_block_fp8_gemm
    status = _launch(args, _raw_stream(index))
    if status:
        N.check(status, "omni_block_fp8_gemm")
    return out


__all__ = ["BlockFp8Rows", "BlockFp8Weight", "block_fp8_linear", "block_fp8_weight",
           "pack_block_fp8", "quantize_block_rows"]
