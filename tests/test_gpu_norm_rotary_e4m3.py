"""Heads turned whole and written to an 8-bit cache in one launch: the scale is of the row that is
written, whatever lanes past the head's last chunk hold. Widths whose chunks are no power of two, both
layouts, factors off one, few tokens and many."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import PagedKvCache, norm_rotary, rotary_frequencies, write_kv_cache

E4M3 = torch.float8_e4m3fn


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("factor", [1.0, 0.5, 1.3])
@pytest.mark.parametrize("dim", [48, 80, 96, 112, 160, 192, 224, 240])
def test_scale_is_of_the_row_that_is_written(gpu, dtype, layout, factor, dim):
    """Every key scale is max|row| / 448 of the key that came out (divided on the CPU, where a division by
    a number is one), and the bytes and scales those of the write on its own."""
    g = torch.Generator().manual_seed(dim)
    inv, _ = rotary_frequencies(dim, device=gpu)
    weight = (1 + 0.3 * torch.randn(dim, generator=g)).to(gpu)
    for tokens in (3, 500, 16000):  # one head a lane group, and four
        qkv = torch.randn(tokens, 6, dim, generator=g).to(dtype).to(gpu)
        q, k, v = qkv.split([2, 2, 2], 1)
        positions = torch.randint(0, 30000, (tokens,), generator=g).to(gpu)
        slots = torch.randperm(tokens + 9, generator=g)[:tokens].to(gpu)
        caches = [PagedKvCache.allocate(-(-(tokens + 9) // 16), 16, 2, dim, E4M3, gpu) for _ in range(2)]
        _, turned = norm_rotary(q, k, positions, inv, q_weight=weight, k_weight=weight, layout=layout,
                                factor=factor, v=v, cache=caches[0], slots=slots)
        held = caches[0].key_scale[slots // 16, :, slots % 16]
        assert torch.equal(held.cpu(), turned.float().abs().amax(2).cpu() / 448)
        write_kv_cache(caches[1], turned, v, slots)
        assert torch.equal(caches[0].key_scale, caches[1].key_scale)
        assert torch.equal(caches[0].value_scale, caches[1].value_scale)
        for a, b in ((caches[0].keys, caches[1].keys), (caches[0].values, caches[1].values)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
