"""Attention of one token over the paged cache against float64: every tile's, wave's and chunk's edges,
pages of any size, grouped heads, 8-bit rows, stale and bad pages, bounds on the lengths, batches,
offsets past 2^32, refusals."""

from __future__ import annotations

import random

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import PagedKvCache, paged_attention

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}
# a softmax weight as the matrix cores take it: two bf16 numbers, or one f16
WEIGHT = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def filled_cache(g, pages, page, kv, dim, held, gpu):
    keys, values = (torch.randn(pages, kv, page, dim, generator=g) for _ in range(2))
    if held is not E4M3:
        return PagedKvCache(keys.to(held).to(gpu), values.to(held).to(gpu))
    values = values * torch.exp(2 * torch.randn(pages, kv, page, 1, generator=g))
    scales = [t.abs().amax(3) / 448 for t in (keys, values)]
    rows = [(t / s[..., None]).to(E4M3).to(gpu) for t, s in zip((keys, values), scales)]
    return PagedKvCache(*rows, *(s.to(gpu) for s in scales))


def table_for(g, lengths, page, pages, gpu, extra=0):
    """A page table of shuffled pages; what lies behind a sequence's pages is out of the cache."""
    columns = max([-(-n // page) for n in lengths] + [0]) + extra
    order = torch.randperm(pages, generator=g, dtype=torch.int64).tolist()
    table = torch.full((len(lengths), columns), 10 ** 9, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for c in range(-(-n // page)):
            table[b, c] = order.pop()
    return table.to(gpu)


def rows_of(cache, table, length):
    """(k, v) [kv_heads, length, dim] in float64."""
    at = torch.arange(length, device=table.device)
    pages, place = table[at // cache.page_size].long(), at % cache.page_size
    out = []
    for t, scale in ((cache.keys, cache.key_scale), (cache.values, cache.value_scale)):
        if scale is None:
            out.append(t[pages, :, place].double().transpose(0, 1))
        else:
            x = t.view(torch.uint8)[pages, :, place].view(E4M3).double()
            out.append((x * scale[pages, :, place].double()[..., None]).transpose(0, 1))
    return out


def check(q, cache, table, lengths, scale=None, **kw):
    """The prompt kernel's bound with this one's weights: scores' relative error twice (weight and sum),
    the weight's own rounding, 16 bits of it twice for 8-bit rows, whose values' scales multiply it first,
    float32 sums over the keys, one rounding."""
    got = paged_attention(q, cache, table, torch.tensor(lengths, dtype=torch.int32, device=q.device),
                          scale=scale, **kw)
    used = q.shape[2] ** -0.5 if scale is None else scale
    group = q.shape[1] // cache.kv_heads
    weight = WEIGHT[torch.bfloat16 if cache.dtype is E4M3 else q.dtype] + 2.0 ** -23
    for b, n in enumerate(lengths):
        if n == 0:
            assert (got[b] == 0).all()
            continue
        k, v = rows_of(cache, table[b], n)
        qs = q[b].double().unflatten(0, (-1, group))
        p = torch.softmax(qs @ k.transpose(1, 2) * used, 2)
        spread = (qs.abs() @ k.abs().transpose(1, 2) * used).amax(2, keepdim=True)
        relative = 2 * ((q.shape[2] + 5) * 2.0 ** -23 * spread + 2.0 ** -22) + n * 2.0 ** -23
        want = (p @ v).flatten(0, 1)
        bound = ((relative + weight) * (p @ v.abs())).flatten(0, 1)
        bound = (bound + HALF_ULP[q.dtype] * want.abs() + TINY[q.dtype]) * (1 + 2.0 ** -7)
        assert ((got[b].double() - want).abs() <= bound).all(), (b, n)
    return got


def queries(g, batch, heads, dim, dtype, gpu, std=2.0):
    return (std * torch.randn(batch, heads, dim, generator=g)).to(dtype).to(gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bytes_held", [False, True])
@pytest.mark.parametrize("heads,kv,dim,page", [(1, 1, 128, 16), (4, 1, 64, 1), (7, 1, 80, 24), (6, 2, 128, 7),
                                               (3, 3, 16, 64), (2, 1, 256, 16), (16, 1, 208, 16),
                                               (20, 1, 64, 32), (40, 1, 48, 5), (32, 8, 128, 256)])
def test_lengths_around_every_edge(gpu, dtype, bytes_held, heads, kv, dim, page):
    g = torch.Generator().manual_seed(heads * dim + page)
    lengths = [1, 0, 31, 32, 33, 15, 127, 128, 129, 160, 255, 256, 257, 511, 513, 1000]
    pages = sum(-(-n // page) for n in lengths) + 3
    cache = filled_cache(g, pages, page, kv, dim, E4M3 if bytes_held else dtype, gpu)
    q = queries(g, len(lengths), heads, dim, dtype, gpu)
    table = table_for(g, lengths, page, pages, gpu)
    got = check(q, cache, table, lengths)
    # a bound on the lengths changes no bit
    assert torch.equal(check(q, cache, table, lengths, max_length=1000), got)


@pytest.mark.parametrize("bytes_held", [False, True])
def test_long_sequences(gpu, bytes_held):
    """Chunks of every size: 2048 and 16384 are the last lengths of 256 and 512."""
    g = torch.Generator().manual_seed(5)
    lengths = [2047, 2048, 2049, 16384, 16385, 40001, 2]
    pages = sum(-(-n // 64) for n in lengths)
    cache = filled_cache(g, pages, 64, 2, 64, E4M3 if bytes_held else torch.bfloat16, gpu)
    q = queries(g, len(lengths), 6, 64, torch.bfloat16, gpu, 4.0)
    check(q, cache, table_for(g, lengths, 64, pages, gpu), lengths)


def test_rows_do_not_depend_on_the_batch(gpu):
    rng, g = random.Random(1), torch.Generator().manual_seed(8)
    lengths = [rng.choice([0, 5, 300, 2000, 9000]) for _ in range(40)]
    pages = sum(-(-n // 16) for n in lengths)
    cache = filled_cache(g, pages, 16, 2, 64, torch.bfloat16, gpu)
    table = table_for(g, lengths, 16, pages, gpu, extra=100)
    q = queries(g, 40, 4, 64, torch.bfloat16, gpu)
    n = torch.tensor(lengths, device=gpu)
    got = paged_attention(q, cache, table, n)
    for b in (0, 7, 39):
        alone = paged_attention(q[b:b + 1], cache, table[b:b + 1], n[b:b + 1], max_length=lengths[b])
        assert torch.equal(alone[0], got[b])
    order = torch.randperm(40, generator=g).to(gpu)
    assert torch.equal(paged_attention(q[order], cache, table[order], n[order].int()), got[order])


@pytest.mark.parametrize("bytes_held", [False, True])
def test_large_and_small_scores(gpu, bytes_held):
    g = torch.Generator().manual_seed(6)
    cache = filled_cache(g, 70, 16, 1, 64, E4M3 if bytes_held else torch.float16, gpu)
    lengths = [1000, 77]
    table = table_for(g, lengths, 16, 70, gpu)
    for std in (0.0, 0.01, 10.0, 60.0):
        q = queries(g, 2, 4, 64, torch.float16, gpu, std)
        check(q, cache, table, lengths)
        check(q, cache, table, lengths, scale=0.02)


@pytest.mark.parametrize("bytes_held", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_stale_rows_do_not_reach_a_query(gpu, bytes_held, bad):
    """What the last page holds behind a sequence's end, and other pages, whatever it is."""
    g = torch.Generator().manual_seed(7)
    cache = filled_cache(g, 30, 24, 2, 64, E4M3 if bytes_held else torch.bfloat16, gpu)
    lengths = [1, 23, 24, 25, 290]
    table = table_for(g, lengths, 24, 30, gpu)
    q = queries(g, 5, 4, 64, torch.bfloat16, gpu)
    want = check(q, cache, table, lengths)
    held = torch.zeros(30, 24, dtype=torch.bool, device=gpu)
    for b, n in enumerate(lengths):
        at = torch.arange(n, device=gpu)
        held[table[b, at // 24].long(), at % 24] = True
    stale = ~held[:, None, :].expand(30, 2, 24)
    if bytes_held:
        cache.keys.view(torch.uint8)[stale] = 0x7f
        cache.values.view(torch.uint8)[stale] = 0x7f
        cache.key_scale[stale], cache.value_scale[stale] = bad, bad
    else:
        cache.keys[stale], cache.values[stale] = bad, bad
    assert torch.equal(check(q, cache, table, lengths), want)


def test_pages_outside_the_cache_are_left_out(gpu):
    g = torch.Generator().manual_seed(9)
    cache = filled_cache(g, 8, 16, 1, 64, torch.bfloat16, gpu)
    q = queries(g, 3, 2, 64, torch.bfloat16, gpu)
    for hole in (-1, 8, 2**31 - 1, -2**31):
        table = torch.tensor([[0, hole, 2], [hole, hole, hole], [3, 4, 5]], dtype=torch.int32, device=gpu)
        n = torch.tensor([40, 48, 48], device=gpu)
        got = paged_attention(q, cache, table, n)
        short = torch.tensor([[2, 0], [3, 4]], dtype=torch.int32, device=gpu)
        assert (got[1] == 0).all()
        # the keys that are left: page 0's 16 and page 2's first 8
        k, v = (t[[0, 2], 0].flatten(0, 1)[:24].double() for t in (cache.keys, cache.values))
        p = torch.softmax(q[0].double() @ k.t() / 8, 1)
        assert ((got[0].double() - p @ v).abs() <= 2.0 ** -7 * (p @ v.abs())).all()
        assert torch.equal(got[2], paged_attention(q, cache, table, n)[2]) and short.numel()


def test_lengths_past_their_bounds(gpu):
    """Lengths below zero are zero, those past the table's room or max_length count as that."""
    g = torch.Generator().manual_seed(10)
    cache = filled_cache(g, 40, 16, 2, 32, torch.bfloat16, gpu)
    q = queries(g, 3, 2, 32, torch.bfloat16, gpu)
    table = torch.randperm(40, generator=g)[:36].view(3, 12).to(torch.int32).to(gpu)
    big = torch.tensor([-7, 2**40, 10**6], device=gpu)
    got = paged_attention(q, cache, table, big)
    assert (got[0] == 0).all()
    assert torch.equal(got[1:], check(q, cache, table, [0, 192, 192])[1:])
    got = paged_attention(q, cache, table, big, max_length=100)
    assert torch.equal(got[1:], check(q, cache, table, [0, 100, 100])[1:])
    assert (paged_attention(q, cache, table, big, max_length=0) == 0).all()
    assert (paged_attention(q, cache, table[:, :0], big) == 0).all()


def test_strides(gpu):
    g = torch.Generator().manual_seed(11)
    keys, values = (torch.randn(9, 16, 4, 64, generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    cache = PagedKvCache(keys.transpose(1, 2), values.transpose(1, 2))  # tokens outside heads
    dense = PagedKvCache(keys.transpose(1, 2).contiguous(), values.transpose(1, 2).contiguous())
    qkv = torch.randn(2, 16 * 64, generator=g).to(torch.bfloat16).to(gpu)
    q = qkv[:, :512].view(2, 8, 64)
    tables = torch.randperm(8, generator=g).view(2, 4).to(torch.int32).to(gpu)
    table = torch.full((2, 9), -1, dtype=torch.int32, device=gpu)
    table[:, 2:6] = tables
    want = check(q.contiguous(), dense, tables, [60, 33])
    assert torch.equal(check(q, cache, table[:, 2:6], [60, 33]), want)
    buffer = torch.full((8, 5, 72), 3.0, dtype=torch.bfloat16, device=gpu)
    out = buffer[:, 1:3, 8:].transpose(0, 1)
    assert torch.equal(check(q, cache, table[:, 2:6], [60, 33], out=out), want)
    assert (buffer[:, [0, 3, 4]] == 3).all() and (buffer[..., :8] == 3).all()


def test_rows_past_two_gigabytes(gpu):
    pages = 2 ** 32 // (64 * 8 * 128) + 40
    cache = PagedKvCache(*(torch.zeros(pages, 8, 64, 128, dtype=torch.bfloat16, device=gpu)
                           for _ in range(2)))
    g = torch.Generator().manual_seed(12)
    for t in (cache.keys, cache.values):
        t[-30:] = torch.randn(30, 8, 64, 128, generator=g).to(torch.bfloat16).to(gpu)
    table = (pages - 1 - torch.randperm(30, generator=g)).view(2, 15).to(torch.int32).to(gpu)
    check(queries(g, 2, 16, 128, torch.bfloat16, gpu), cache, table, [960, 501])


def test_no_rows_and_refusals(gpu):
    cache = PagedKvCache.allocate(4, 16, 2, 64, torch.bfloat16, gpu)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device=gpu)
    table = torch.zeros(3, 2, dtype=torch.int32, device=gpu)
    n = torch.zeros(3, dtype=torch.int32, device=gpu)
    assert paged_attention(q[:0], cache, table[:0], n[:0]).shape == (0, 4, 64)
    wide = torch.zeros(3, 4, 68, dtype=torch.bfloat16, device=gpu)
    for args, kw in [((q.float(), cache, table, n), {}), ((q.half(), cache, table, n), {}),
                     ((q[..., :32], cache, table, n), {}), ((q[:, :3], cache, table, n), {}),
                     ((q[0], cache, table, n), {}), ((wide[..., :64], cache, table, n), {}),
                     ((q, cache, table.long(), n), {}), ((q, cache, table[:2], n), {}),
                     ((q, cache, table[0], n), {}), ((q, cache, table.t().contiguous().t(), n), {}),
                     ((q, cache, table, n[:2]), {}), ((q, cache, table, n.float()), {}),
                     ((q, cache, table, n.repeat(2)[::2]), {}), ((q, cache, table, n), {"scale": -1.0}),
                     ((q, cache, table, n), {"max_length": -1}), ((q, cache, table, n), {"out": q[:2]}),
                     ((q, cache, table, n), {"out": q.half()})]:
        with pytest.raises(ValueError):
            paged_attention(*args, **kw)
    with pytest.raises(N.OmniCodecError):
        paged_attention(q.cpu(), cache, table, n)
