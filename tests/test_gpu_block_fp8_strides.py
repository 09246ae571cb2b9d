"""8-bit linear layers on operands that lie gigabytes apart: float rows, as the last tokens of a long
padded batch, and the blocks' scales of very many rows."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import (BlockFp8Rows, block_fp8_linear, pack_block_fp8,
                                     quantize_block_rows)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 2, 16, 17])
def test_float_rows_gigabytes_apart(gpu, rows):
    g = torch.Generator().manual_seed(rows)
    k, stride = 1040, 2**30 // 7 if rows > 2 else 2**31 + 8  # elements: offsets past 32 bits
    w = pack_block_fp8(torch.randn(96, k, generator=g)).to(gpu)
    x = torch.randn(rows, k, generator=g).to(torch.bfloat16).to(gpu)
    buffer = torch.empty((rows - 1) * stride + k, dtype=torch.bfloat16, device=gpu)
    apart = buffer.as_strided((rows, k), (stride, 1))
    apart.copy_(x)
    assert torch.equal(block_fp8_linear(apart, w), block_fp8_linear(x, w))


@pytest.mark.parametrize("rows,n", [(5, 40), (40, 96), (300, 1300), (700, 1301), (1030, 1300),
                                    (2050, 1029), (3500, 4360)])
@pytest.mark.parametrize("blocks", [1, 2, 3])
def test_block_scales_gigabytes_apart(gpu, rows, n, blocks):
    """Block-major scales whose blocks lie 2^29 bytes apart: the stages that a tile reads ahead end
    past the last block, 32 bits of offset further on."""
    g = torch.Generator(device=gpu).manual_seed(rows)
    w = pack_block_fp8(torch.randn(n, 128 * blocks, generator=g, device=gpu))
    q = quantize_block_rows(torch.randn(rows, 128 * blocks, generator=g, device=gpu))
    apart = torch.empty((blocks - 1) * 2**27 + rows, device=gpu).as_strided((rows, blocks), (1, 2**27))
    apart.copy_(q.scale)
    for out in (torch.bfloat16, torch.float32):
        assert torch.equal(block_fp8_linear(BlockFp8Rows(q.values, apart), w, out_dtype=out),
                           block_fp8_linear(q, w, out_dtype=out))
