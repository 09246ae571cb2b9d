"""The stated accuracy of the 8-bit linear layers where products cancel: bf16 outputs within what the
8-bit matrix instruction may cut from each group of 8 features, f32 outputs within float32 sums."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import BlockFp8Rows, BlockFp8Weight, block_fp8_linear

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _any(g, *shape):
    """Any finite E4M3 values, zeros and subnormals among them."""
    bits = torch.randint(0, 256, shape, generator=g).to(torch.uint8)
    bits[(bits & 0x7f) == 0x7f] = 0
    return bits.view(E4M3).float()


def _expanded(scale, per_row, rows, cols):
    return scale.double().repeat_interleave(per_row, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def _check(x, w):
    """x [rows, k], w [n, k] scaled E4M3 operands against float64 on the CPU: the cut of every aligned
    8 features, up to (k + 8) steps of 2^-23 of the terms' magnitudes, and one rounding to the type."""
    got16 = block_fp8_linear(x, w).cpu().double()
    got32 = block_fp8_linear(x, w, out_dtype=torch.float32).cpu().double()
    (rows, k), n = x.values.shape, w.weight.shape[0]
    a, b = x.values.cpu().double(), w.weight.cpu().double()
    sa, sb = _expanded(x.scale.cpu(), 1, rows, k), _expanded(w.scale.cpu(), 128, n, k)
    want, size = (a * sa) @ (b * sb).T, (a * sa).abs() @ (b * sb).abs().T
    low = 2.0 ** -6
    ca, cb = a.abs().clamp_min(low) * sa, b.abs().clamp_min(low) * sb
    cut = torch.zeros(rows, n, dtype=torch.float64)
    for f in range(0, k, 8):
        cut += 7 * 2.0 ** -13 * (ca[:, None, f:f + 8] * cb[None, :, f:f + 8]).amax(2)
    steps = (k + 8) * 2.0 ** -23 * size + 2.0 ** -25
    assert ((got32 - want).abs() <= steps + 2.0 ** -24 * want.abs()).all()
    assert ((got16 - want).abs() <= cut + steps + 2.0 ** -8 * (want.abs() + cut + steps)).all()


@pytest.mark.parametrize("rows", [1, 16, 40, 300])
def test_cancelling_products(gpu, rows):
    """Three quarters of the features in pairs whose products cancel exactly; the rest is the result."""
    g = torch.Generator().manual_seed(rows)
    k, n = 400, 140
    x, w = _any(g, rows, k), _any(g, n, k)
    pair = torch.rand(k // 2, generator=g) < 0.75
    x.view(rows, -1, 2)[:, pair, 1] = x.view(rows, -1, 2)[:, pair, 0]
    w.view(n, -1, 2)[:, pair, 1] = -w.view(n, -1, 2)[:, pair, 0]
    x[:, 5::7] *= 2.0 ** -6  # rounded to E4M3 again below: many subnormals and zeros
    scales = torch.rand(rows, 4, generator=g) + 0.1, torch.rand(2, 4, generator=g) + 0.1
    _check(BlockFp8Rows(x.to(E4M3).to(gpu), scales[0].to(gpu)),
           BlockFp8Weight(w.to(E4M3).to(gpu), scales[1].to(gpu)))


@pytest.mark.parametrize("rows", [1, 40])
def test_small_beside_cancelling(gpu, rows):
    """256 - 256 + a small product in one group of 8: a bf16 output keeps it down to 2^-13 of 256 (to
    the bit, a power of two), an f32 output always."""
    k, n = 128, 9
    x, w = torch.zeros(rows, k), torch.zeros(n, k)
    x[:, 0] = x[:, 1] = 256
    x[:, 2] = 0.25
    w[:, 0], w[:, 1] = 1, -1
    w[:, 2] = 2.0 ** -torch.arange(n)
    small = 0.25 * w[0:, 2].expand(rows, n)
    rows8 = BlockFp8Rows(x.to(E4M3).to(gpu), torch.ones(rows, 1, device=gpu))
    weight = BlockFp8Weight(w.to(E4M3).to(gpu), torch.ones(1, 1, device=gpu))
    assert torch.equal(block_fp8_linear(rows8, weight, out_dtype=torch.float32).cpu(), small)
    kept = small >= 2.0 ** -13 * 256
    got = block_fp8_linear(rows8, weight).cpu().float()
    assert torch.equal(got[kept], small[kept])
    assert ((got - small).abs() <= 7 * 2.0 ** -13 * 256).all()
