"""The context operators together: prompts in pieces, then token after token, over one cache; in a
captured graph and on a side stream; and the example that runs them from text to audio."""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest
import torch

from sglang_omni_amd.kernels import (PagedKvCache, norm_rotary, paged_attention, prompt_attention,
                                     read_kv_cache, rotary_frequencies)

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _starts(lengths, gpu):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=gpu)


def _attention64(q, k, v):
    """q [heads, dim] over k, v [kv_heads, length, dim], in float64; and the sum of its parts' sizes."""
    group = q.shape[0] // k.shape[0]
    p = torch.softmax(q.double().unflatten(0, (-1, group)) @ k.double().transpose(1, 2)
                      * q.shape[1] ** -0.5, 2)
    return (p @ v.double()).flatten(0, 1), (p @ v.double().abs()).flatten(0, 1)


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("dim", [64, 80])
def test_pieces_and_steps_over_one_cache(gpu, held, dim):
    """Two pieces of three prompts, then steps: every output against float64 over the keys and values
    that the cache stands for. Off by half a bf16 step of the weights and one of the result, and a tenth of
    that for the float32 sums (the scores' own rounding: (dim + 4) 2^-22 of their parts, below 2^-12)."""
    g = torch.Generator().manual_seed(dim)
    heads, kv, page = 6, 2, 16
    inv, _ = rotary_frequencies(dim, device=gpu)
    weight = (1 + 0.2 * torch.randn(dim, generator=g)).to(gpu)
    cache = PagedKvCache.allocate(64, page, kv, dim, held, gpu)
    table = torch.randperm(63, generator=g).view(3, 21).to(gpu)
    lengths = [0, 0, 0]

    def slots_of(stream, start, end):
        at = torch.arange(start, end, device=gpu)
        return table[stream, at // page] * page + at % page

    def layer(counts):
        """The next `counts` tokens of each stream: their q, outputs of norm_rotary with the cache."""
        n = sum(counts)
        qkv = torch.randn(n, heads + 2 * kv, dim, generator=g).to(torch.bfloat16).to(gpu)
        q, k, v = qkv.split([heads, kv, kv], 1)
        positions = torch.cat([torch.arange(b, b + c) for b, c in zip(lengths, counts)]).to(gpu)
        slots = torch.cat([slots_of(s, b, b + c) for s, (b, c) in enumerate(zip(lengths, counts))])
        q, k = norm_rotary(q, k, positions, inv, q_weight=weight, k_weight=weight, v=v, cache=cache,
                           slots=slots)
        for s, c in enumerate(counts):
            lengths[s] += c
        return q, k, v

    def check(out, q, counts):
        row = 0
        for s, c in enumerate(counts):
            k, v = (t.float().transpose(0, 1) for t in
                    read_kv_cache(cache, slots_of(s, 0, lengths[s]), dtype=torch.float32))
            for i in range(c):
                m = lengths[s] - c + 1 + i
                want, size = _attention64(q[row], k[:, :m], v[:, :m])
                bound = 2.0 ** -8 * 1.1 * size + 2.0 ** -8 * want.abs()
                assert ((out[row].double() - want).abs() <= bound).all()
                row += 1

    counts = [17, 40, 1]
    q, k, v = layer(counts)
    out = prompt_attention(q, k, v, _starts(counts, gpu))
    if held is not E4M3:  # the cache holds what the first piece's attention read
        check(out, q, counts)
    counts = [30, 5, 64]
    q, k, v = layer(counts)
    whole = torch.cat([slots_of(s, 0, lengths[s]) for s in range(3)])
    keys, values = read_kv_cache(cache, whole, dtype=torch.bfloat16)
    out = prompt_attention(q, keys, values, _starts(counts, gpu), key_starts=_starts(lengths, gpu))
    if held is not E4M3:  # 8-bit rows are read back as bf16, rounded once more
        check(out, q, counts)
    for _ in range(4):
        q, k, v = layer([1, 1, 1])
        out = paged_attention(q, cache, table.int(), torch.tensor(lengths, device=gpu))
        check(out, q, [1, 1, 1])


@pytest.mark.parametrize("held", [torch.bfloat16, E4M3])
def test_captured_in_a_graph_and_on_a_side_stream(gpu, held):
    """A decode step and a prompt captured once each, replayed on other inputs between eager work, each
    graph with its own workspace; and the same on a stream that is not the default one."""
    g = torch.Generator().manual_seed(3)
    heads, kv, dim, batch, page = 8, 2, 64, 5, 16
    inv, _ = rotary_frequencies(dim, device=gpu)
    cache = PagedKvCache.allocate(batch * 200, page, kv, dim, held, gpu)
    table = torch.randperm(batch * 200, generator=g).view(batch, 200).to(torch.int32).to(gpu)
    qkv = torch.zeros(batch, heads + 2 * kv, dim, dtype=torch.bfloat16, device=gpu)
    positions = torch.zeros(batch, dtype=torch.int64, device=gpu)
    prompt = torch.zeros(300, heads + 2 * kv, dim, dtype=torch.bfloat16, device=gpu)
    starts = _starts([100, 50, 150], gpu)

    def decode():
        slots = table[torch.arange(batch, device=gpu), positions // page].long() * page + positions % page
        q, k, v = qkv.split([heads, kv, kv], 1)
        q, k = norm_rotary(q, k, positions, inv, v=v, cache=cache, slots=slots)
        return paged_attention(q, cache, table, positions + 1)

    def whole():
        q, k, v = prompt.split([heads, kv, kv], 1)
        q, k = norm_rotary(q, k, torch.arange(300, device=gpu), inv)
        few = prompt_attention(q[:7], k, v, torch.tensor([0, 7], dtype=torch.int32, device=gpu)
                               if not torch.cuda.is_current_stream_capturing() else few_starts,
                               key_starts=few_keys)
        return prompt_attention(q, k, v, starts), few

    few_starts = torch.tensor([0, 7], dtype=torch.int32, device=gpu)
    few_keys = torch.tensor([0, 300], dtype=torch.int32, device=gpu)

    def refill(k):
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        prompt.copy_(torch.randn(prompt.shape, generator=g))
        positions.copy_(torch.randint(0, 200 * page, (batch,), generator=g))
        cache.keys.view(torch.uint8).copy_(
            torch.randint(0, 60, cache.keys.view(torch.uint8).shape, generator=g, dtype=torch.uint8))

    refill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            aside = decode(), *whole()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(aside, (decode(), *whole())))
    graphs, held_out = [], []
    for f in (decode, whole):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held_out.append(f())
        graphs.append(graph)
    for k in range(4):
        refill(k)
        want = decode(), *whole()
        torch.cuda.synchronize()
        for graph in graphs[::-1] if k % 2 else graphs:
            graph.replay()
        torch.cuda.synchronize()
        got = held_out[0], *held_out[1]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location(
        "talker_context", Path(__file__).resolve().parents[1] / "examples" / "talker_context.py")
    module = importlib.util.module_from_spec(spec)
    sys.modules["talker_context"] = module
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_example_from_text_to_audio(gpu, example, cache):
    from sglang_omni_amd.models import DacCodecDecoder, DacDecoderConfig, make_dac_weights

    config = example.ContextTalkerConfig()
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, config.text_vocab, (n,), generator=g).tolist() for n in (3, 50, 200)]

    def talker():
        return example.ContextTalker(config, 4, 80, gpu, cache_dtype=example.CACHES[cache])

    first = talker()
    codes = first.codes(prompts, 6)
    assert codes.shape == (3, 4, 6) and int(codes.min()) >= 0 and int(codes.max()) < config.codebook_size
    assert first.lengths == [3 + 23, 50 + 23, 200 + 23, 0]
    assert torch.equal(talker().codes(prompts, 6), codes)
    for s in range(3):
        first.release(s)
    assert sorted(first.free) == list(range(80))
    # a prompt in two pieces: what came before is read back from the cache
    pieces = talker()
    pieces.prompt([p[:2] for p in prompts], [0, 1, 2])
    logits = pieces.prompt([p[2:] for p in prompts], [0, 1, 2])
    assert logits.shape == (3, config.vocab) and logits.isfinite().all()
    assert pieces.lengths == [3, 50, 200, 0]
    codec = DacDecoderConfig(n_codebooks=4, codebook_size=256, latent_dim=64, channels=128, rates=(2, 4))
    audio = DacCodecDecoder(make_dac_weights(codec, seed=0), codec, device=gpu).from_indices(codes)
    assert audio.shape == (3, 1, 6 * codec.hop_length) and audio.isfinite().all()
