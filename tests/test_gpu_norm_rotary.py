"""Head norms with rotary positions, alone and into the paged cache, and the cache's rows there and
back: against float64, every head width's split, strides, slots outside the cache, 8-bit rows bit for
bit, refusals."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import (PagedKvCache, apply_rotary, norm_rotary, read_kv_cache,
                                     rotary_frequencies, write_kv_cache)

E4M3 = torch.float8_e4m3fn
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def _exact(t, weight, eps, positions, inv_freq, layout, factor):
    """The result in float64, and the size of what each value is a sum of."""
    v = t.double()
    n = v / (v.pow(2).mean(2, keepdim=True) + eps).sqrt()
    if weight is not None:
        n = n * weight.double()
    angle = positions.double()[:, None] * inv_freq
    c, s = angle.cos()[:, None] * factor, angle.sin()[:, None] * factor
    pairs = inv_freq.shape[0]
    i = torch.arange(pairs, device=t.device)
    a_at, b_at = (i, i + pairs) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = n[..., a_at], n[..., b_at]
    out, size = n.clone(), n.abs()
    size[..., a_at] = size[..., b_at] = (a.abs() + b.abs()) * factor
    out[..., a_at], out[..., b_at] = a * c - b * s, b * c + a * s
    return out, size


def _check(got, t, weight, eps, positions, inv_freq, layout, factor):
    """The sum of dim squares, all of one sign, is within dim 2^-24 of itself, its root within half
    that; quotient, root, mean, eps and two products add 6 * 2^-24; sine and cosine within 2^-22, two
    products and a sum; then one rounding to the type."""
    want, size = _exact(t, weight, eps, positions, inv_freq, layout, factor)
    relative = t.shape[2] * 2.0 ** -25 + 6 * 2.0 ** -24 + 2.0 ** -21
    bound = relative * size * (1 + HALF_ULP[t.dtype]) + HALF_ULP[t.dtype] * want.abs() + TINY[t.dtype]
    assert got.dtype == t.dtype
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (128, 128), (128, 64), (80, 80), (80, 40), (96, 32),
                                            (256, 256), (512, 512), (70, 70), (66, 2), (24, 12), (5, 4),
                                            (2, 2), (511, 2), (512, 6)])
def test_heads(gpu, dtype, layout, dim, rotary_dim):
    g = torch.Generator().manual_seed(dim + rotary_dim)
    inv, _ = rotary_frequencies(rotary_dim, 1e4, device=gpu)
    weights = [(1 + 0.3 * torch.randn(dim, generator=g)).to(gpu) for _ in range(2)]
    for tokens, heads, kv in ((1, 1, 1), (1, 16, 8), (7, 3, 2), (130, 5, 1), (4000, 9, 3)):
        if tokens * dim > 4000 * 128:
            continue
        qkv = 3 * torch.randn(tokens, (heads + 2 * kv) * dim + 3, generator=g)
        qkv = qkv.to(dtype).to(gpu)
        q = qkv[:, 1:1 + heads * dim].unflatten(1, (heads, dim))  # a view off the 16-byte grid
        k = qkv[:, 1 + heads * dim:1 + (heads + kv) * dim].unflatten(1, (kv, dim))
        positions = torch.randint(-5, 200000, (tokens,), generator=g).to(gpu)
        qo, ko = norm_rotary(q, k, positions, inv, q_weight=weights[0], k_weight=weights[1], eps=1e-5,
                             layout=layout, factor=1.25)
        _check(qo, q, weights[0], 1e-5, positions, inv, layout, 1.25)
        _check(ko, k, weights[1], 1e-5, positions, inv, layout, 1.25)
        alone = norm_rotary(q, None, positions.int(), inv, eps=1e-5, layout=layout, factor=1.25)
        _check(alone, q, None, 1e-5, positions, inv, layout, 1.25)


@pytest.mark.gpu
def test_hard_rows(gpu):
    """Rows of zeros stay zero, tiny rows are what eps makes of them, a NaN or an infinity spoils its
    own head alone."""
    inv, _ = rotary_frequencies(64, device=gpu)
    q = torch.randn(6, 3, 64, generator=torch.Generator().manual_seed(1)).to(gpu)
    q[0, 1] = 0
    q[1] *= 1e-18
    q[2, 0, 5], q[3, 2, 63] = float("nan"), float("inf")
    positions = torch.arange(6, device=gpu)
    got = norm_rotary(q, None, positions, inv, eps=1e-6)
    assert (got[0, 1] == 0).all()
    rest = torch.ones(6, 3, dtype=torch.bool, device=gpu)
    rest[2, 0] = rest[3, 2] = False
    assert got[rest].isfinite().all() and got[2, 0].isnan().all()
    for t in (0, 1, 4, 5):
        _check(got[t:t + 1], q[t:t + 1], None, 1e-6, positions[t:t + 1], inv, "half", 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_and_strided_outputs(gpu, layout):
    g = torch.Generator().manual_seed(4)
    inv, _ = rotary_frequencies(48, device=gpu)
    qkv = torch.randn(33, 6 * 64, generator=g).to(torch.bfloat16).to(gpu)
    q, k = qkv[:, :256].view(33, 4, 64), qkv[:, 256:].view(33, 2, 64)
    positions = torch.arange(66, device=gpu)[::2]
    want = norm_rotary(q, k, positions, inv, layout=layout)
    buffer = torch.full((2, 4, 33, 64), float("nan"), dtype=torch.bfloat16, device=gpu)
    out = (buffer[0].transpose(0, 1), buffer[1, :2].transpose(0, 1))  # heads outside tokens
    got = norm_rotary(q, k, positions, inv, layout=layout, q_out=out[0], k_out=out[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert buffer[1, 2:].isnan().all()
    norm_rotary(q, k, positions, inv, layout=layout, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def _quantized(rows):
    """Rows' E4M3 bytes and scales by their definition, on the CPU."""
    x = rows.float().cpu()
    amax = x.abs().amax(-1, keepdim=True)
    tiny, most = amax < 2.0 ** -100, torch.full_like(amax, 448.0)
    q = (x * torch.where(tiny, torch.ones_like(amax), most / amax)).to(E4M3)
    return q.view(torch.uint8), torch.where(tiny, torch.ones_like(amax), amax / most)[..., 0]


def _held(cache, slots):
    """The cache's rows and scales at slots: bytes of E4M3."""
    page, place = slots // cache.page_size, slots % cache.page_size
    rows = [t.view(torch.uint8) if cache.dtype is E4M3 else t for t in (cache.keys, cache.values)]
    rows = [t[page, :, place].cpu() for t in rows]
    if cache.dtype is E4M3:
        rows += [t[page, :, place].cpu() for t in (cache.key_scale, cache.value_scale)]
    return rows


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("held", [torch.bfloat16, torch.float16, E4M3])
@pytest.mark.parametrize("page,kv,dim", [(1, 1, 16), (16, 8, 128), (24, 3, 80), (64, 2, 256), (7, 5, 48)])
def test_write_and_read(gpu, dtype, held, page, kv, dim):
    g = torch.Generator().manual_seed(page + dim)
    for tokens in (1, 5, 333):
        pages = -(-tokens // page) + 2
        cache = PagedKvCache.allocate(pages, page, kv, dim, held, gpu)
        before = cache.keys.clone()
        k, v = (torch.randn(tokens, kv, dim, generator=g) * torch.rand(tokens, kv, 1, generator=g)
                for _ in range(2))
        k[0, 0] = 0
        kv_rows = torch.cat([k, v], 1).to(dtype).to(gpu)
        k, v = kv_rows[:, :kv], kv_rows[:, kv:]
        slots = torch.randperm(pages * page, generator=g)[:tokens].to(gpu)
        write_kv_cache(cache, k, v, slots if tokens != 5 else slots.int())
        got = _held(cache, slots)
        if held is E4M3:
            want = [_quantized(k), _quantized(v)]
            assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[1][0])
            assert torch.equal(got[2], want[0][1]) and torch.equal(got[3], want[1][1])
            values = [(b.view(E4M3).float() * s[..., None]) for b, s in want]
        else:
            assert torch.equal(got[0], k.to(held).cpu()) and torch.equal(got[1], v.to(held).cpu())
            values = [got[0].float(), got[1].float()]
        touched = torch.zeros(pages * page, dtype=torch.bool)
        touched[slots.cpu()] = True
        same = (cache.keys.view(torch.uint8) == before.view(torch.uint8)).all(3).all(1).flatten().cpu()
        assert same[~touched].all()
        for as_type in (torch.bfloat16, torch.float16, torch.float32):
            back = read_kv_cache(cache, slots, dtype=as_type)
            assert all(torch.equal(b.cpu(), w.to(as_type)) for b, w in zip(back, values))


@pytest.mark.gpu
def test_slots_outside_the_cache(gpu):
    """Padded tokens write nothing and read as zeros, whatever their index."""
    cache = PagedKvCache.allocate(3, 4, 2, 32, torch.bfloat16, gpu)
    cache.keys.fill_(7), cache.values.fill_(9)
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(7, 2, 32, generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    slots = torch.tensor([-1, 12, 5, 2**31, -2**40, 11, 2**32 + 5], device=gpu)
    write_kv_cache(cache, k, v, slots)
    back = read_kv_cache(cache, slots)
    for b, t in zip(back, (k, v)):
        assert torch.equal(b[[2, 5]], t[[2, 5]]) and (b[[0, 1, 3, 4, 6]] == 0).all()
    untouched = torch.ones(12, dtype=torch.bool, device=gpu)
    untouched[[5, 11]] = False
    assert (cache.keys.transpose(1, 2).flatten(0, 1)[untouched] == 7).all()
    assert (cache.values.transpose(1, 2).flatten(0, 1)[untouched] == 9).all()


@pytest.mark.gpu
def test_hard_rows_in_8_bits(gpu):
    """Zeros and rows below 2^-100 hold zeros with scale 1; NaN stays and leaves the scale to the
    others; an infinity spoils its own row."""
    cache = PagedKvCache.allocate(1, 8, 1, 16, E4M3, gpu)
    k = torch.ones(5, 1, 16, device=gpu)
    k[0] = 0
    k[1] = 2.0 ** -101
    k[2, 0, 3] = float("nan")
    k[3, 0, 3] = float("inf")
    k[4] *= 3.3e38
    slots = torch.arange(5, device=gpu)
    write_kv_cache(cache, k, k, slots)
    back, _ = read_kv_cache(cache, slots, dtype=torch.float32)
    assert (back[0] == 0).all() and (back[1] == 0).all() and (cache.key_scale[0, 0, :2] == 1).all()
    assert back[2, 0, 3].isnan() and (back[2, 0, :3] == 1).all() and (back[2, 0, 4:] == 1).all()
    assert back[3].isnan().all()
    assert torch.allclose(back[4], k[4], rtol=2.0 ** -4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("held", [torch.bfloat16, torch.float16, E4M3])
@pytest.mark.parametrize("dim,rotary_dim", [(128, 128), (80, 40), (64, 24), (32, 10)])
def test_one_launch_is_norm_rotation_and_write(gpu, dtype, held, dim, rotary_dim):
    """The same bits as three calls one after the other, in either order of tokens and heads."""
    g = torch.Generator().manual_seed(dim)
    inv, _ = rotary_frequencies(rotary_dim, device=gpu)
    weight = (1 + 0.3 * torch.randn(dim, generator=g)).to(gpu)
    for tokens in (3, 700, 9000):
        qkv = torch.randn(tokens, 10 * dim, generator=g).to(dtype).to(gpu)
        q, k, v = qkv.view(tokens, 10, dim).split([4, 3, 3], 1)
        positions = torch.randint(0, 5000, (tokens,), generator=g).to(gpu)
        slots = torch.randperm(tokens + 20, generator=g)[:tokens].to(gpu)
        slots[tokens // 2] = -1
        caches = [PagedKvCache.allocate(-(-(tokens + 20) // 16), 16, 3, dim, held, gpu) for _ in range(2)]
        want = norm_rotary(q, k, positions, inv, q_weight=weight, k_weight=weight)
        write_kv_cache(caches[0], want[1], v, slots)
        got = norm_rotary(q, k, positions, inv, q_weight=weight, k_weight=weight, v=v, cache=caches[1],
                          slots=slots)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        for a, b in ((caches[0].keys, caches[1].keys), (caches[0].values, caches[1].values)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        if held is E4M3:
            assert torch.equal(caches[0].key_scale, caches[1].key_scale)
            assert torch.equal(caches[0].value_scale, caches[1].value_scale)


@pytest.mark.gpu
def test_pages_with_tokens_outside_heads(gpu):
    """[pages, page_size, kv_heads, dim] storage as a transposed view, and a cache that is a part of a
    larger one."""
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(40, 3, 32, generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    slots = torch.randperm(48, generator=g)[:40].to(gpu)
    storage = torch.zeros(2, 6, 8, 5, 32, dtype=torch.bfloat16, device=gpu)
    cache = PagedKvCache(*(t[:, :, 1:4].transpose(1, 2) for t in storage))
    write_kv_cache(cache, k, v, slots)
    assert torch.equal(storage[0, :, :, 1:4].flatten(0, 1)[slots], k)
    assert (storage[:, :, :, [0, 4]] == 0).all()
    back = read_kv_cache(cache, slots)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)


@pytest.mark.gpu
def test_rows_past_two_gigabytes(gpu):
    """Slots whose bytes and elements lie past 2^32."""
    pages = (2 ** 32 // (64 * 8 * 128)) + 100
    cache = PagedKvCache(*(torch.empty(pages, 8, 64, 128, dtype=torch.bfloat16, device=gpu)
                           for _ in range(2)))
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn(200, 8, 128, generator=g).to(torch.bfloat16).to(gpu) for _ in range(2))
    slots = torch.arange(pages * 64 - 200, pages * 64, device=gpu)
    write_kv_cache(cache, k, v, slots)
    back = read_kv_cache(cache, slots)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    assert torch.equal(cache.keys[-1, :, -1], k[-1])


@pytest.mark.gpu
def test_no_tokens_and_refusals(gpu):
    inv, _ = rotary_frequencies(32, device=gpu)
    q = torch.zeros(5, 2, 64, device=gpu)
    at = torch.arange(5, device=gpu)
    cache = PagedKvCache.allocate(2, 4, 2, 64, torch.bfloat16, gpu)
    assert norm_rotary(q[:0], None, at[:0], inv).shape == (0, 2, 64)
    write_kv_cache(cache, q[:0], q[:0], at[:0])
    assert read_kv_cache(cache, at[:0])[0].shape == (0, 2, 64)
    weight = torch.ones(64, device=gpu)
    into = {"v": q, "cache": cache, "slots": at}
    for args, kw in [((q.double(), None, at, inv), {}), ((q[0], None, at, inv), {}),
                     ((q.transpose(1, 2), None, at, inv), {}), ((q, None, at[:4], inv), {}),
                     ((q, None, at.float(), inv), {}), ((q, None, at, inv.float()), {}),
                     ((q[..., :30], None, at, inv), {}), ((q, q[:4], at, inv), {}),
                     ((q, q.half(), at, inv), {}), ((q, None, at, inv), {"layout": "neox"}),
                     ((q, None, at, inv), {"k_out": q}), ((q, None, at, inv), {"q_out": q[:4]}),
                     ((q, None, at, inv), {"q_weight": weight.half()}),
                     ((q, None, at, inv), {"q_weight": weight[:32]}),
                     ((q, None, at, inv), {"eps": -1.0}), ((q, None, at, inv), into),
                     ((q, q, at, inv), {**into, "v": q[:4]}), ((q, q, at, inv), {**into, "v": None}),
                     ((q, q, at, inv), {**into, "slots": at[:4]}),
                     ((q, q, at, inv), {**into, "slots": at.float()}),
                     ((q, q, at, inv), {"slots": at}), ((q, q[:, :1], at, inv), into),
                     ((torch.zeros(5, 1, 514, device=gpu), None, at, inv), {})]:
        with pytest.raises(ValueError):
            norm_rotary(*args, **kw)
    with pytest.raises(N.OmniCodecError):
        norm_rotary(q.cpu(), None, at, inv)
    for args in ((q, q[:4], at), (q, q.half(), at), (q[:, :1], q[:, :1], at), (q, q, at[:4]),
                 (q.long(), q.long(), at)):
        with pytest.raises(ValueError):
            write_kv_cache(cache, *args)
    with pytest.raises(N.OmniCodecError):
        write_kv_cache(cache, q.cpu(), q.cpu(), at)
    for kw in ({"dtype": torch.int32}, {"k_out": q, "v_out": q.half()}, {"k_out": q[:4], "dtype": torch.float32}):
        with pytest.raises(ValueError):
            read_kv_cache(cache, at, **kw)
    with pytest.raises(ValueError):
        read_kv_cache(cache, at.float())
    rows = torch.zeros(2, 2, 4, 64, dtype=torch.bfloat16, device=gpu)
    scale = torch.ones(2, 2, 4, device=gpu)
    for args in ((rows, rows[..., :32]), (rows[..., :24], rows[..., :24]), (rows.float(), rows.float()),
                 (rows[0], rows[0]), (rows.transpose(2, 3), rows.transpose(2, 3)), (rows, rows, scale, scale),
                 (rows.view(torch.uint8).view(E4M3), rows.view(torch.uint8).view(E4M3)),
                 (rows[:0], rows[:0]), (rows.flatten()[1:-63].view(-1, 1, 1, 64)[:2],) * 2):
        with pytest.raises(ValueError):
            PagedKvCache(*args)
    with pytest.raises(N.OmniCodecError):
        PagedKvCache(rows.cpu(), rows.cpu())


@pytest.mark.gpu
def test_rotary_alone_is_what_it_was(gpu):
    """apply_rotary shares the sine and cosine."""
    inv, _ = rotary_frequencies(64, device=gpu)
    q = torch.randn(9, 2, 64, generator=torch.Generator().manual_seed(2)).to(gpu)
    positions = torch.arange(9, device=gpu) * 1000
    unit = q / (q.double().pow(2).mean(2, keepdim=True) + 1e-30).sqrt()
    a = apply_rotary(unit.float(), None, positions, inv).double()
    b = norm_rotary(q, None, positions, inv, eps=1e-30).double()
    assert ((a - b).abs() <= (64 * 2.0 ** -25 + 2.0 ** -20) * unit.abs().amax(2, keepdim=True) * 2).all()
