"""8-bit linear layers on float rows that lie gigabytes apart, as the last tokens of a long padded
batch do."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import block_fp8_linear, pack_block_fp8

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
