"""What the other tests of the context operators run without looking at: the sequence beside one with
holes in its pages, a prompt over the rows of an 8-bit cache, the keys that the example's next piece of
a prompt reads back."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import (PagedKvCache, norm_rotary, paged_attention, prompt_attention,
                                     read_kv_cache, rotary_frequencies)
from tests.test_gpu_paged_attention import check as check_paged, filled_cache, queries
from tests.test_gpu_prompt_attention import check as check_prompt, exact
from tests.test_gpu_talker_context import example  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("hole", [-1, 80, 2**31 - 1, -2**31])
def test_beside_a_sequence_with_holes(gpu, held, hole):
    """One chunk and several: the intact sequence has the bits of a call without holes, and float64's value."""
    g = torch.Generator().manual_seed(19)
    cache = filled_cache(g, 80, 16, 1, 64, held, gpu)
    q = queries(g, 3, 2, 64, torch.bfloat16, gpu)
    whole = torch.stack([torch.randperm(80, generator=g)[:40] for _ in range(3)]).to(torch.int32).to(gpu)
    for lengths in ([40, 48, 48], [600, 640, 630]):
        table = whole.clone()
        table[0, 1], table[1] = hole, hole
        want = check_paged(q, cache, whole, lengths)
        lengths_gpu = torch.tensor(lengths, device=gpu)
        got = paged_attention(q, cache, table, lengths_gpu)
        assert torch.equal(got[2], want[2]) and (got[1] == 0).all()
        # the first one: its other keys, packed on pages of their own
        left = torch.cat([whole[0, :1], whole[0, 2:]])[None].contiguous()
        alone, bound = (paged_attention(q[:1], cache, left, lengths_gpu[:1] - 16),
                        2 * 2.0 ** -8 * 1.01 * cache_most(cache))
        assert ((got[:1].double() - alone.double()).abs() <= bound).all()


def cache_most(cache):
    """The largest value held: an output, of weights that sum to one, is off by half a bf16 step of it (and 2^-16
    for the weights) at most, in either of two orders of the keys."""
    values = cache.values.view(torch.uint8).view(E4M3).float() * cache.value_scale[..., None] \
        if cache.dtype is E4M3 else cache.values.float()
    return values.abs().max().item()


@pytest.mark.parametrize("dim", [64, 80, 128])
def test_a_prompt_over_an_8_bit_cache(gpu, dim):
    """Two pieces; the second over everything read back as bf16, as float64 has it over the same rows; the rows
    are those of their scales and bytes, and within an E4M3 step of the keys that went in."""
    g = torch.Generator().manual_seed(dim)
    heads, kv, page = 6, 2, 16
    inv, _ = rotary_frequencies(dim, device=gpu)
    cache = PagedKvCache.allocate(40, page, kv, dim, E4M3, gpu)
    table = torch.randperm(39, generator=g).view(3, 13).to(gpu)
    lengths, pieces = [0, 0, 0], ([17, 40, 1], [30, 5, 64])
    given = [[] for _ in range(3)]
    for counts in pieces:
        n = sum(counts)
        q, k, v = torch.randn(n, heads + 2 * kv, dim, generator=g).to(torch.bfloat16).to(gpu) \
            .split([heads, kv, kv], 1)
        positions = torch.cat([torch.arange(b, b + c) for b, c in zip(lengths, counts)]).to(gpu)
        stream = torch.repeat_interleave(torch.arange(3), torch.tensor(counts)).to(gpu)
        slots = table[stream, positions // page] * page + positions % page
        q, k = norm_rotary(q, k, positions, inv, v=v, cache=cache, slots=slots)
        for s, (a, b) in enumerate(zip(k.split(counts), v.split(counts))):
            given[s].append((a, b))
            lengths[s] += counts[s]
    at = [torch.arange(n, device=gpu) for n in lengths]
    whole = torch.cat([table[s, a // page] * page + a % page for s, a in enumerate(at)])
    keys, values = read_kv_cache(cache, whole, dtype=torch.bfloat16)
    for i, back in enumerate((keys, values)):
        want = torch.cat([t[i] for rows in given for t in rows]).float()
        # half an E4M3 step of the value (or of 2^-6, the least normal one, in steps of the scale), one of bf16
        scale = want.abs().amax(2, keepdim=True) / 448
        bound = (2.0 ** -4 * want.abs()).clamp(min=0) + 2.0 ** -10 * 1.01 * scale + 2.0 ** -8 * 1.07 * want.abs()
        assert ((back.float() - want).abs() <= bound * (1 + 2.0 ** -10)).all()
    check_prompt(q, keys, values, list(pieces[1]), lengths)


@pytest.mark.parametrize("held", ["bf16", "e4m3"])
def test_the_examples_next_piece_reads_what_came_before(gpu, example, monkeypatch, held):  # noqa: F811
    """Its first layer's keys are those of the prompt in one piece, at their own positions, bit for bit from a
    16-bit cache and as the cache rounds them from an 8-bit one; its attention is float64's over them."""
    config = example.ContextTalkerConfig()
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, config.text_vocab, (n,), generator=g).tolist() for n in (3, 50, 200)]
    calls = []

    def recorded(q, k, v, starts, *, key_starts=None):
        out = prompt_attention(q, k, v, starts, key_starts=key_starts)
        calls.append((q, k, v, starts, key_starts, out))
        return out

    monkeypatch.setattr(example, "prompt_attention", recorded)

    def talker():
        return example.ContextTalker(config, 4, 80, gpu, cache_dtype=example.CACHES[held])

    whole = talker()
    whole.prompt(prompts, [0, 1, 2])
    one = calls[0]
    calls.clear()
    pieces, cuts = talker(), [2, 20, 77]
    pieces.prompt([p[:c] for p, c in zip(prompts, cuts)], [0, 1, 2])
    calls.clear()
    pieces.prompt([p[c:] for p, c in zip(prompts, cuts)], [0, 1, 2])
    q, k, v, starts, key_starts, out = calls[0]
    ends = [0, 3, 53, 253]
    counts = [n - c for n, c in zip((3, 50, 200), cuts)]
    assert key_starts.tolist() == ends and starts.tolist() == [0, *torch.tensor(counts).cumsum(0).tolist()]
    assert torch.equal(q, torch.cat([one[0][e + c:f] for e, c, f in zip(ends, cuts, ends[1:])]))
    for got, want in ((k, one[1]), (v, one[2])):
        if held == "bf16":
            assert torch.equal(got, want)
        else:
            scale = want.float().abs().amax(2, keepdim=True) / 448
            bound = (2.0 ** -4 + 2.0 ** -8 * 1.07) * want.float().abs() + 2.0 ** -10 * 1.01 * scale
            assert ((got.float() - want.float()).abs() <= bound * (1 + 2.0 ** -10)).all()
    want, bound = exact(q, k, v, counts, [3, 50, 200], True, config.head_dim ** -0.5)
    assert ((out.double() - want).abs() <= bound).all()
