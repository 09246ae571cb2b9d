"""NaN in what a query of paged attention sees is NaN in its output, in one chunk of keys and in
several; a row whose scores are all -infinity is zero; neither reaches another row or head."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import PagedKvCache, paged_attention

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def cache_of(g, gpu, pages, kv, dim, dtype):
    keys, values = (torch.randn(pages, kv, 16, dim, generator=g).to(gpu) for _ in range(2))
    if dtype is not E4M3:
        return PagedKvCache(keys.to(dtype), values.to(dtype))
    return PagedKvCache(keys.to(E4M3), values.to(E4M3),
                        *(torch.ones(pages, kv, 16, device=gpu) for _ in range(2)))


@pytest.mark.parametrize("dtype,held", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                        (torch.bfloat16, E4M3), (torch.float16, E4M3)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("length", [1, 300, 512, 513, 3000, 20000])
def test_a_query_of_nan(gpu, dtype, held, dim, length):
    g = torch.Generator().manual_seed(length + dim)
    pages = -(-length // 16)
    cache = cache_of(g, gpu, pages, 2, dim, held)
    table = torch.arange(pages, dtype=torch.int32, device=gpu).expand(3, pages)
    lengths = torch.tensor([length] * 3, device=gpu)
    q = torch.randn(3, 4, dim, generator=g).to(dtype).to(gpu)
    clean = paged_attention(q, cache, table, lengths)
    assert clean.isfinite().all()
    q[1, 2, 7] = float("nan")
    got = paged_attention(q, cache, table, lengths)
    assert got[1, 2].isnan().all()
    # its group's other head shares its waves' maxima: off by two roundings at most, of weights and result,
    # on either side; all other rows keep their bits
    off = (got[1, 3].double() - clean[1, 3].double()).abs()
    values = cache.values.float().abs().max().item()
    assert (off <= 4 * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) * values).all()
    got[1, 2:] = clean[1, 2:]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("length,first,last", [(300, 0, 300), (300, 64, 96), (3000, 256, 512), (3000, 1, 2999),
                                               (3000, 0, 3000), (20000, 512, 1024), (20000, 19999, 20000)])
def test_keys_of_nan(gpu, held, length, first, last):
    """Keys first .. last - 1 of one head, whole tiles and chunks among them."""
    g = torch.Generator().manual_seed(length + first)
    pages = -(-length // 16)
    cache = cache_of(g, gpu, pages, 2, 64, held)
    table = torch.randperm(pages, generator=g).to(torch.int32)[None].to(gpu)
    lengths = torch.tensor([length], device=gpu)
    q = torch.randn(1, 6, 64, generator=g).to(torch.bfloat16).to(gpu)
    clean = paged_attention(q, cache, table, lengths)
    at = torch.arange(first, last, device=gpu)
    page, place = table[0, at // 16].long(), at % 16
    if held is E4M3:
        cache.keys.view(torch.uint8)[page, 1, place] = 0x7f
    else:
        cache.keys[page, 1, place] = float("nan")
    got = paged_attention(q, cache, table, lengths)
    assert torch.equal(got[:, :3], clean[:, :3]) and got[:, 3:].isnan().all()


@pytest.mark.parametrize("length", [40, 512, 513, 3000])
@pytest.mark.parametrize("value", [1.0, float("inf"), float("nan")])
def test_scores_of_minus_infinity(gpu, length, value):
    """All of a row's scores -infinity: zero, in one chunk and in several, whatever the values are."""
    g = torch.Generator().manual_seed(length)
    pages = -(-length // 16)
    cache = cache_of(g, gpu, pages, 1, 64, torch.bfloat16)
    cache.keys[..., 5] = float("-inf")
    cache.values[..., 9] = value
    q = torch.rand(1, 2, 64, generator=g).to(torch.bfloat16).to(gpu) + 0.5
    table = torch.arange(pages, dtype=torch.int32, device=gpu)[None]
    got = paged_attention(q, cache, table, torch.tensor([length], device=gpu))
    assert (got == 0).all()
