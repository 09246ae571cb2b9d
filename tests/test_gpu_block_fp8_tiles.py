"""Every tile of the 8-bit linear layers over many K blocks, past 64 of them (a register's worth of
weight scales) and past 128, with a partial last block and scales of very different sizes; the larger
tiles also on strided and padded operands, unaligned outputs, non-finite and float rows, and again and
again. The sizes lie well inside the range where a tile is estimated fastest."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import (BlockFp8Rows, BlockFp8Weight, block_fp8_linear,
                                     quantize_block_rows)

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
# rows and columns that the tiles take on 256 CUs: 16 rows; 32 x 32, 32 x 64, 64 x 64, 64 x 128,
# 128 x 128 and 256 x 256 (128 x 128 with f32 output)
FEW = (16, 530)
SMALL = [(100, 2000), (300, 1300), (700, 1301)]
LARGE = [(1030, 1300), (2050, 1029), (3500, 4360)]


def _operands(gpu, rows, k, n, seed):
    """Random E4M3 values without NaN, and scales over 2^-6 .. 2^6, no two blocks' alike."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    blocks = -(-k // 128)

    def values(r):
        return torch.randn(r, k, generator=g, device=gpu).mul_(64).clamp_(-448, 448).to(E4M3)

    def scales(r):
        return torch.exp2(12 * torch.rand(r, blocks, generator=g, device=gpu) - 6)

    return (BlockFp8Rows(values(rows), scales(rows)),
            BlockFp8Weight(values(n), scales(-(-n // 128)),
                           torch.randn(n, generator=g, device=gpu)))


def _expanded(scale, per_row, rows, cols):
    return scale.double().repeat_interleave(per_row, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _check_f32(y, x, w):
    """k products and k / 128 scaled blocks, each step within 2^-23 of the terms' magnitudes, the
    bias and one rounding."""
    a = x.values.double() * _expanded(x.scale, 1, *x.values.shape)
    b = w.weight.double() * _expanded(w.scale, 128, *w.weight.shape)
    want = a @ b.T + w.bias.double()
    size = a.abs_() @ b.abs_().T + w.bias.double().abs()
    assert ((y.double() - want).abs() <= (x.values.shape[1] + 8) * 2.0 ** -23 * size).all()


@pytest.mark.parametrize("k", [2064, 8208, 12304, 16400])
@pytest.mark.parametrize("rows,n", [FEW, *SMALL, *LARGE])
def test_many_blocks(gpu, rows, n, k):
    """f32 outputs against float64, and bf16 ones against the same rows 16 at a time (one order of the
    blocks everywhere; those 16 against float64 in the tests of the bound)."""
    x, w = _operands(gpu, rows, k, n, rows + k)
    _check_f32(block_fp8_linear(x, w, out_dtype=torch.float32), x, w)
    whole = block_fp8_linear(x, w)
    if rows > 16:
        for at in (0, 16, rows // 2, rows - 16):
            part = BlockFp8Rows(x.values[at:at + 16], x.scale[at:at + 16])
            assert torch.equal(block_fp8_linear(part, w), whole[at:at + 16])
    for _ in range(3):
        assert torch.equal(block_fp8_linear(x, w), whole)


@pytest.mark.parametrize("rows,n", LARGE)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_larger_tiles_strided(gpu, rows, n, out):
    """Rows and weights as slices with NaN bytes on every side, block-major scales, an output off every
    alignment, whose surroundings stay."""
    k = 2064
    x, w = _operands(gpu, rows, k, n, rows)
    want = block_fp8_linear(x, w, out_dtype=out)

    def padded(t):
        wide = torch.full((t.shape[0] + 3, k + 304), 0x7f, dtype=torch.uint8, device=gpu)
        inner = wide[1:-2, 160:160 + k]
        inner.copy_(t.view(torch.uint8))
        return wide.view(E4M3)[1:-2, 160:160 + k]

    buffer = torch.full((rows + 1, n + 10), float("nan"), dtype=out, device=gpu)
    got = block_fp8_linear(BlockFp8Rows(padded(x.values), x.scale.t().contiguous().t()),
                           BlockFp8Weight(padded(w.weight), w.scale, w.bias),
                           buffer[:rows, 3:n + 3])
    assert torch.equal(got, want)
    assert buffer[rows].isnan().all() and buffer[:, :3].isnan().all() and buffer[:, n + 3:].isnan().all()


@pytest.mark.parametrize("rows,n", LARGE)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_larger_tiles_non_finite(gpu, rows, n, out):
    """A NaN value, an infinite scale and a NaN weight spoil their row or column alone."""
    x, w = _operands(gpu, rows, 1040, n, rows + 1)
    clean = block_fp8_linear(x, w, out_dtype=out)
    x.values.view(torch.uint8)[7, 1000] = 0x7f
    x.scale[rows - 1, 3] = float("inf")
    w.weight.view(torch.uint8)[n - 2, 0] = 0xff
    got = block_fp8_linear(x, w, out_dtype=out)
    assert got[7].isnan().all() and got[:, n - 2].isnan().all()
    assert not got[rows - 1].isfinite().any()
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[7], rest[rows - 1], rest[:, n - 2] = False, False, False
    assert torch.equal(got[rest], clean[rest])


@pytest.mark.parametrize("rows,n", LARGE)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_larger_tiles_float_rows(gpu, rows, n, dtype):
    _, w = _operands(gpu, 1, 2064, n, rows + 2)
    g = torch.Generator(device=gpu).manual_seed(rows)
    x = torch.randn(rows, 2070, generator=g, device=gpu).to(dtype)[:, 3:2063]  # 2 060 features, odd start
    for out in (torch.bfloat16, torch.float32):
        assert torch.equal(block_fp8_linear(x, w, out_dtype=out),
                           block_fp8_linear(quantize_block_rows(x), w, out_dtype=out))
