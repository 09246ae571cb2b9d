"""Packing linear weights to 8 bits where some are not finite, on the CPU."""

from __future__ import annotations

import torch

from sglang_omni_amd.kernels import pack_block_fp8


def test_nan_stays_its_own():
    """A NaN weight is NaN; the others of its block keep their scale and values."""
    w = torch.randn(130, 300, generator=torch.Generator().manual_seed(0)) * 0.02
    clean = pack_block_fp8(w)
    w[5, 7], w[129, 299] = float("nan"), float("nan")
    before = torch.where(w.isnan(), 0.0, w)  # the scales that the other weights have
    got, want = pack_block_fp8(w), pack_block_fp8(before)
    assert torch.equal(got.scale, want.scale) and got.scale.shape == clean.scale.shape
    nan = torch.zeros(130, 304, dtype=torch.bool)
    nan[5, 7] = nan[129, 299] = True
    assert torch.equal(got.weight.float().isnan(), nan)
    assert torch.equal(got.weight.float()[~nan], want.weight.float()[~nan])


def test_infinity_spoils_its_block():
    """As in the row quantizer: an infinite scale, so that every product with the block is NaN."""
    w = torch.randn(130, 300, generator=torch.Generator().manual_seed(1))
    clean = pack_block_fp8(w)
    w[3, 200] = -float("inf")
    got = pack_block_fp8(w)
    assert got.scale[0, 1] == float("inf")
    rest = torch.ones(2, 3, dtype=torch.bool)
    rest[0, 1] = False
    assert torch.equal(got.scale[rest], clean.scale[rest])
    full = got.weight.float() * got.scale.repeat_interleave(128, 0)[:130].repeat_interleave(128, 1)[:, :304]
    assert full[:128, 128:256].isnan().all()
