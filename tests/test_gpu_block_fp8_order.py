"""A row's bits in the 8-bit linear layers do not depend on the rows beside it: one token, a decode
batch and a prefill add an element's K blocks in one order, whichever kernel and tile takes them, and
float rows give the bits of the same rows quantized before."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import (BlockFp8Rows, block_fp8_linear, pack_block_fp8,
                                     quantize_block_rows)

pytestmark = pytest.mark.gpu


def _operands(gpu, rows, k, n, seed, bias=True):
    g = torch.Generator().manual_seed(seed)
    # blocks of very different sizes: another order of the sum is another result
    size = torch.exp2(torch.randint(-6, 7, (-(-k // 128),), generator=g).float())
    x = torch.randn(rows, k, generator=g) * size.repeat_interleave(128)[:k]
    w = torch.randn(n, k, generator=g) / k ** 0.5
    return x.to(gpu), pack_block_fp8(w, torch.randn(n, generator=g) if bias else None).to(gpu)


# 1 to 130 K blocks: less than a round of the few-row kernel's waves, several, and past 64 and 128
@pytest.mark.parametrize("k", [112, 1040, 2064, 4096, 8208, 16400])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_few_rows_are_the_bits_of_many(gpu, k, out):
    x, w = _operands(gpu, 300, k, 530, k)
    q = quantize_block_rows(x)
    whole = block_fp8_linear(q, w, out_dtype=out)
    for rows in (1, 2, 15, 16, 17, 40):
        for at in (0, 300 - rows):
            part = BlockFp8Rows(q.values[at:at + rows], q.scale[at:at + rows])
            assert torch.equal(block_fp8_linear(part, w, out_dtype=out), whole[at:at + rows])


@pytest.mark.parametrize("k", [100, 1040, 4096, 8208])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_float_rows_are_the_bits_of_quantized_ones(gpu, k, dtype):
    x, w = _operands(gpu, 40, k, 200, k + 1)
    x = x.to(dtype)
    for out in (torch.bfloat16, torch.float32):
        whole = block_fp8_linear(quantize_block_rows(x), w, out_dtype=out)
        for rows in (1, 3, 16, 17, 40):
            assert torch.equal(block_fp8_linear(x[:rows], w, out_dtype=out), whole[:rows])
