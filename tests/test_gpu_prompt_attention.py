"""Attention of packed prompts against float64: every tile's edges, grouped heads, lengths of zero,
queries that see nothing, strides, infinities and NaN where a query does not look, rows behind the last
sequence, refusals."""

from __future__ import annotations

import itertools
import random

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import prompt_attention

pytestmark = pytest.mark.gpu

HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}
TINY = {torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def starts_of(lengths, gpu, dtype=torch.int32):
    return torch.tensor([0, *itertools.accumulate(lengths)], dtype=dtype, device=gpu)


def exact(q, k, v, lengths, key_lengths, causal, scale):
    """(result in float64, bound on what an output may be off).

    A score is a sum of dim exact products in float32: off by dim * 2^-23 of the sum of their sizes, its
    product with the scale, the difference to the maximum and the exponential by 4 * 2^-23 of the largest
    score and 2^-22 more. So a weight is relatively off by twice that (numerator and maximum's cancel in
    the quotient, the denominator has its own), by half a step of the type, and by the float32 sums over
    the keys; each product of it with a value is off by as much of itself. Then one rounding."""
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    group = q.shape[1] // k.shape[1]
    at = key_at = 0
    for n, m in zip(lengths, key_lengths):
        for h in range(q.shape[1]):
            qs, ks = q[at:at + n, h].double(), k[key_at:key_at + m, h // group].double()
            vs = v[key_at:key_at + m, h // group].double()
            scores = qs @ ks.t() * scale
            sizes = qs.abs() @ ks.abs().t() * scale
            if causal:
                hidden = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(m - n + 1)
                scores.masked_fill_(hidden, -torch.inf)
                sizes.masked_fill_(hidden, 0)
            if m == 0:
                continue
            p = torch.softmax(scores, 1)
            p[(scores == -torch.inf).all(1)] = 0
            spread = sizes.amax(1, keepdim=True)
            relative = 2 * ((q.shape[2] + 4) * 2.0 ** -23 * spread + 2.0 ** -22) + m * 2.0 ** -23
            # what is hidden counts nothing, whatever it holds
            seen = torch.where((p > 0).any(0)[:, None], vs, 0.0)
            o = p @ seen
            out[at:at + n, h] = o
            bound[at:at + n, h] = ((relative + HALF_ULP[q.dtype]) * (p @ seen.abs())
                                   + HALF_ULP[q.dtype] * o.abs() + TINY[q.dtype]) * (1 + 2.0 ** -7)
        at, key_at = at + n, key_at + m
    return out, bound


def check(q, k, v, lengths, key_lengths=None, causal=True, scale=None, **kw):
    key_lengths = lengths if key_lengths is None else key_lengths
    given = None if key_lengths is lengths else starts_of(key_lengths, q.device)
    got = prompt_attention(q, k, v, starts_of(lengths, q.device), key_starts=given, causal=causal,
                           scale=scale, **kw)
    want, bound = exact(q, k, v, lengths, key_lengths, causal,
                        q.shape[2] ** -0.5 if scale is None else scale)
    total = sum(lengths)
    assert got.shape == q.shape and got.dtype == q.dtype
    assert ((got[:total].double() - want[:total]).abs() <= bound[:total]).all()
    return got


def random_heads(g, tokens, heads, dim, dtype, gpu, std=1.0):
    return (std * torch.randn(tokens, heads, dim, generator=g)).to(dtype).to(gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 128), (4, 1, 64), (7, 1, 80), (6, 2, 128), (8, 8, 8),
                                          (2, 2, 256), (3, 1, 200), (40, 2, 64), (16, 8, 128), (5, 5, 40)])
def test_lengths_around_every_tile(gpu, dtype, causal, heads, kv, dim):
    g = torch.Generator().manual_seed(heads * dim)
    for lengths in ([1], [31, 32, 33], [63, 64, 65, 1], [127, 0, 128, 129], [0, 0, 5, 0], [300, 17, 0],
                    [255, 256, 257]):
        t = sum(lengths)
        q = random_heads(g, t, heads, dim, dtype, gpu, 2.0)
        k, v = (random_heads(g, t, kv, dim, dtype, gpu) for _ in range(2))
        check(q, k, v, lengths, causal=causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_queries_and_keys_of_their_own_lengths(gpu, dtype, causal):
    """Later pieces of longer sequences; fewer keys than queries leave the first queries nothing to
    see; no keys at all."""
    g = torch.Generator().manual_seed(9)
    lengths, key_lengths = [5, 70, 64, 1, 130, 3, 40], [900, 70, 30, 513, 0, 2, 41]
    q = random_heads(g, sum(lengths), 4, 64, dtype, gpu)
    k, v = (random_heads(g, sum(key_lengths), 2, 64, dtype, gpu) for _ in range(2))
    got = check(q, k, v, lengths, key_lengths, causal=causal)
    assert (got[140:270] == 0).all() == True  # the sequence without keys
    if causal:
        assert (got[75:75 + 34] == 0).all() and (got[270] == 0).all()


def test_one_long_sequence(gpu):
    g = torch.Generator().manual_seed(11)
    q = random_heads(g, 3001, 4, 128, torch.bfloat16, gpu, 3.0)
    k, v = (random_heads(g, 3001, 2, 128, torch.bfloat16, gpu) for _ in range(2))
    check(q, k, v, [3001])
    check(q, k, v, [3001], causal=False)
    check(q[:100], k, v, [100], [3001])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("lengths,before,heads,kv,rows,split", [
    ([700, 650], 0, 64, 16, 128, False), ([300], 0, 4, 2, 32, False), ([500], 15000, 32, 4, 128, True),
    ([3], 6000, 4, 2, 32, True), ([9, 0, 31], 3000, 8, 2, 32, True)])
def test_every_form(gpu, dtype, dim, lengths, before, heads, kv, rows, split):
    """Rows of a workgroup 32 or 128, the keys of a row in one piece or several."""
    key_lengths = [n + before for n in lengths]
    tile = N.ctypes.c_int()
    pieces = N.load_library().omni_prompt_plan(sum(lengths), sum(key_lengths), len(lengths), heads, kv, dim,
                                               1, N.ctypes.byref(tile))
    assert (pieces > 1) == split and tile.value == rows
    g = torch.Generator().manual_seed(dim + before)
    q = random_heads(g, sum(lengths), heads, dim, dtype, gpu, 2.0)
    k, v = (random_heads(g, sum(key_lengths), kv, dim, dtype, gpu) for _ in range(2))
    check(q, k, v, lengths, key_lengths)
    # rows behind the last sequence, and a sequence whose queries see nothing
    few = [*lengths[:-1], lengths[-1] - 2]
    got = check(q, k, v, few, key_lengths)
    assert (got[sum(few):] == 0).all()
    out = torch.full_like(q, 7.0)
    prompt_attention(q, k, v, starts_of(few, gpu), key_starts=starts_of(key_lengths, gpu), out=out)
    assert torch.equal(out[:sum(few)], got[:sum(few)]) and (out[sum(few):] == 7).all()


def test_many_sequences(gpu):
    """More than a search step's 64 and than 64 * 64, empty ones among them."""
    rng = random.Random(3)
    lengths = [rng.choice([0, 0, 1, 1, 2, 3]) for _ in range(4500)] + [70]
    g = torch.Generator().manual_seed(2)
    t = sum(lengths)
    q = random_heads(g, t, 2, 16, torch.bfloat16, gpu)
    k, v = (random_heads(g, t, 1, 16, torch.bfloat16, gpu) for _ in range(2))
    got = check(q, k, v, lengths)
    assert torch.equal(got, prompt_attention(q, k, v, starts_of(lengths, gpu, torch.int64)))
    for few in (lengths[:65], lengths[:150]):
        check(q[:sum(few)], k[:sum(few)], v[:sum(few)], few)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_and_small_scores(gpu, dtype):
    """Scores of hundreds, a row that looks at one key alone, maxima that grow and fall along the keys,
    and another scale."""
    g = torch.Generator().manual_seed(21)
    for std in (0.0, 0.01, 10.0, 40.0):
        q = random_heads(g, 333, 2, 64, dtype, gpu, std)
        k, v = (random_heads(g, 333, 2, 64, dtype, gpu) for _ in range(2))
        check(q, k, v, [333])
        ramp = torch.linspace(0, 4, 333, device=gpu)[:, None, None]
        check(q, (k * ramp).to(dtype), v, [333], causal=False)
        check(q, (k * ramp.flip(0)).to(dtype), v, [333], scale=0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("heads,dim", [(1, 64), (4, 128), (2, 256)])
def test_what_a_query_does_not_see_does_not_reach_it(gpu, dtype, bad, heads, dim):
    g = torch.Generator().manual_seed(31)
    lengths = [100, 37, 150]
    q = random_heads(g, 287, heads, dim, dtype, gpu)
    k, v = (random_heads(g, 287, 1, dim, dtype, gpu) for _ in range(2))
    clean = prompt_attention(q, k, v, starts_of(lengths, gpu))
    for at in (60, 99, 100, 136, 137, 137 + 70, 286):
        first = 0 if at < 100 else 100 if at < 137 else 137
        last = 100 if at < 100 else 137 if at < 137 else 287
        for spoil_key in (False, True):
            k2, v2 = k.clone(), v.clone()
            v2[at, 0, 3] = bad
            if spoil_key:
                k2[at] = bad
            got = prompt_attention(q, k2, v2, starts_of(lengths, gpu))
            unaware = torch.ones(287, dtype=torch.bool, device=gpu)
            unaware[at:last] = False
            assert got[unaware].isfinite().all()
            assert torch.equal(got[:first], clean[:first]) and torch.equal(got[last:], clean[last:])
            # the same sums, in another order where the tile is taken key by key
            want, bound = exact(q[first:at], k[first:at], v[first:at], [at - first], [at - first], True,
                                dim ** -0.5)
            assert ((got[first:at].double() - want).abs() <= bound).all()
            if not spoil_key:
                assert not got[at:last, :, 3].isfinite().any()
                others = [d for d in range(dim) if d != 3]
                want, bound = exact(q[first:last], k[first:last], v[first:last], [last - first],
                                    [last - first], True, dim ** -0.5)
                off = (got[first:last].double() - want).abs()
                assert (off[..., others] <= bound[..., others]).all()


def test_rows_behind_the_last_sequence(gpu):
    g = torch.Generator().manual_seed(41)
    q = random_heads(g, 200, 4, 64, torch.bfloat16, gpu)
    k, v = (random_heads(g, 200, 2, 64, torch.bfloat16, gpu) for _ in range(2))
    q[130:], k[130:], v[130:] = float("nan"), float("nan"), float("inf")
    for lengths in ([100, 30], [130], [0, 130, 0]):
        got = check(q, k, v, lengths)
        assert (got[130:] == 0).all()
        out = torch.full_like(q, 7.0)
        prompt_attention(q, k, v, starts_of(lengths, gpu), out=out)
        assert torch.equal(out[:130], got[:130]) and (out[130:] == 7).all()
    assert (prompt_attention(q, k, v, starts_of([], gpu)) == 0).all()
    assert (prompt_attention(q, k, v, starts_of([0, 0], gpu)) == 0).all()


def test_strides(gpu):
    """Views of a qkv buffer, heads outside tokens, keys shared by an expanded head, a strided output."""
    g = torch.Generator().manual_seed(51)
    lengths = [90, 71]
    qkv = torch.randn(161, 8 * 64 + 16, generator=g).to(torch.bfloat16).to(gpu)
    q, k, v = qkv[:, 8:520].unflatten(1, (8, 64)).split([4, 2, 2], 1)
    want = prompt_attention(q.contiguous(), k.contiguous(), v.contiguous(), starts_of(lengths, gpu))
    buffer = torch.full((4, 170, 80), 5.0, dtype=torch.bfloat16, device=gpu)
    out = buffer[:, 3:164, 8:72].transpose(0, 1)
    got = prompt_attention(q, k, v, starts_of(lengths, gpu), out=out)
    assert got is out and torch.equal(got, want)
    assert (buffer[:, :3] == 5).all() and (buffer[:, 164:] == 5).all() and (buffer[..., 72:] == 5).all()
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    assert torch.equal(prompt_attention(*turned, starts_of(lengths, gpu)), want)
    one = k[:, :1]
    got = prompt_attention(q, one.expand(161, 2, 64), v, starts_of(lengths, gpu))
    assert torch.equal(got, prompt_attention(q, one.repeat(1, 2, 1), v, starts_of(lengths, gpu)))


def test_neighbours_values_do_not_matter(gpu):
    """The same bits beside other sequences' other values."""
    g = torch.Generator().manual_seed(61)
    lengths = [77, 300, 5]
    for heads, kv in ((6, 3), (64, 32)):
        q = random_heads(g, 382, heads, 128, torch.bfloat16, gpu)
        k, v = (random_heads(g, 382, kv, 128, torch.bfloat16, gpu) for _ in range(2))
        got = prompt_attention(q, k, v, starts_of(lengths, gpu))
        for t in (q, k, v):
            t[:77] *= 3
            t[377:] = float("nan")
        again = prompt_attention(q, k, v, starts_of(lengths, gpu))
        assert torch.equal(got[77:377], again[77:377])


def test_no_tokens_and_refusals(gpu):
    q = torch.zeros(8, 4, 64, dtype=torch.bfloat16, device=gpu)
    k = torch.zeros(8, 2, 64, dtype=torch.bfloat16, device=gpu)
    s = starts_of([8], gpu)
    assert prompt_attention(q[:0], k[:0], k[:0], starts_of([], gpu)).shape == (0, 4, 64)
    assert prompt_attention(q, k[:0], k[:0], s, key_starts=starts_of([0], gpu)).eq(0).all()
    wide = torch.zeros(8, 4, 68, dtype=torch.bfloat16, device=gpu)
    for args, kw in [((q.float(), k.float(), k.float(), s), {}), ((q, k.half(), k, s), {}),
                     ((q, k, k[:4], s), {}), ((q, k[..., :32], k[..., :32], s), {}),
                     ((q[:, :3], k, k, s), {}), ((q, k[:, :0], k[:, :0], s), {}), ((q[0], k, k, s), {}),
                     ((q.transpose(1, 2), k, k, s), {}), ((wide[..., :64], k, k, s), {}),
                     ((wide[..., 4:], k, k, s), {}), ((q, k, k, s.float()), {}), ((q, k, k, s[0]), {}),
                     ((q, k, k, s[:0]), {}), ((q, k, k, s), {"key_starts": s[:1]}),
                     ((q, k, k, s), {"key_starts": s.long()}), ((q, k, k, s), {"scale": 0.0}),
                     ((q, k, k, s), {"scale": float("nan")}), ((q, k, k, s), {"out": q[:4]}),
                     ((q, k, k, s), {"out": q.half()}),
                     ((torch.zeros(8, 1, 264, dtype=torch.bfloat16, device=gpu),) * 3 + (s,), {})]:
        with pytest.raises(ValueError):
            prompt_attention(*args, **kw)
    with pytest.raises(ValueError):
        prompt_attention(q, k, k, s.cpu())
    with pytest.raises(N.OmniCodecError):
        prompt_attention(q.cpu(), k.cpu(), k.cpu(), s.cpu())


def test_starts_that_are_not_ascending_stay_inside(gpu):
    """Starts out of range are clamped: whatever they say, no row outside is read or written."""
    g = torch.Generator().manual_seed(71)
    q = random_heads(g, 64, 2, 64, torch.bfloat16, gpu)
    k, v = (random_heads(g, 64, 1, 64, torch.bfloat16, gpu) for _ in range(2))
    want = prompt_attention(q, k, v, starts_of([64], gpu))
    for values in ([-5, 64], [0, 900], [-2**31, 2**31 - 1]):
        got = prompt_attention(q, k, v, torch.tensor(values, dtype=torch.int32, device=gpu))
        assert torch.equal(got, want)
    got = prompt_attention(q, k, v, torch.tensor([0, 40, 10, 64], dtype=torch.int32, device=gpu))
    assert got.shape == q.shape
