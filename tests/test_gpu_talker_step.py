"""The talker example: the 8-bit operators together, from tokens to audio."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from sglang_omni_amd.kernels import (adjust_logits, apply_rotary, block_fp8_linear,
                                     gated_residual_norm, pack_block_fp8, rotary_frequencies)
from sglang_omni_amd.models import DacCodecDecoder, DacDecoderConfig, make_dac_weights

pytestmark = pytest.mark.gpu

_SPEC = importlib.util.spec_from_file_location(
    "talker_step", Path(__file__).resolve().parents[1] / "examples" / "talker_step.py")


@pytest.fixture(scope="module")
def example():
    import sys

    module = importlib.util.module_from_spec(_SPEC)
    sys.modules["talker_step"] = module
    _SPEC.loader.exec_module(module)
    return module


def _dense(w):
    full = w.scale.repeat_interleave(128, 0)[:w.weight.shape[0]].repeat_interleave(128, 1)
    return w.weight.float() * full[:, :w.weight.shape[1]]


def _rms(v, weight, eps):
    return v * torch.rsqrt(v.pow(2).mean(1, keepdim=True) + eps) * weight


def _first_logits(talker, tokens):
    """A stream's first token attends to itself alone: every head returns its value row."""
    c = talker.config
    h = talker.embedding[tokens].float()
    for layer in talker.layers:
        v = (_rms(h, layer.norms[0], c.eps) @ _dense(layer.qkv).T)[:, -c.kv_heads * c.head_dim:]
        v = v.view(-1, c.kv_heads, 1, c.head_dim).expand(-1, -1, c.heads // c.kv_heads, -1).flatten(1)
        h = h + layer.scales[0] * _rms(v @ _dense(layer.o).T, layer.norms[1], c.eps)
        gate, up = (_rms(h, layer.norms[2], c.eps) @ _dense(layer.gate_up).T).chunk(2, 1)
        y = (torch.nn.functional.silu(gate) * up) @ _dense(layer.down).T
        h = h + layer.scales[1] * _rms(y, layer.norms[3], c.eps)
    return _rms(h, talker.final_norm, c.eps) @ _dense(talker.head).T


@pytest.mark.parametrize("streams", [1, 5, 40])
def test_first_token_against_plain_torch(gpu, example, streams):
    """float32 torch with the same dequantized weights. Only the activations' 8-bit rounding differs:
    a uniform error of up to 2^-4 of a value is 2^-4 / sqrt(3) = 3.6 % of it in the mean square, four
    products a layer behind norms that keep its share; 2 layers and the head stay under 3.6 % * 3 =
    sqrt(9) of them."""
    talker = example.Talker(example.TalkerConfig(), streams, gpu)
    tokens = torch.arange(streams, device=gpu) * 7
    rows = talker.hidden_rows(tokens, torch.arange(streams, device=gpu))
    got = block_fp8_linear(rows, talker.head, out_dtype=torch.float32)
    want = _first_logits(talker, tokens)
    assert ((got - want).norm() / want.norm()).item() <= 0.036 * 3


def test_codes_follow_their_codebooks_and_decode(gpu, example):
    config = example.TalkerConfig()
    talker = example.Talker(config, 6, gpu)
    codes = talker.codes(5, 25)  # 100 positions: past the 72-frame window
    assert codes.shape == (5, 4, 25) and int(codes.min()) >= 0
    assert int(codes.max()) < config.codebook_size
    assert torch.equal(talker.lengths.cpu(), torch.tensor([100] * 5 + [0], dtype=torch.int32))
    assert torch.equal(talker.positions.cpu(), torch.tensor([100] * 5 + [0]))
    again = example.Talker(config, 6, gpu).codes(5, 25)
    assert torch.equal(codes, again)
    alone = example.Talker(config, 6, gpu)  # a stream's codes do not depend on its neighbours
    assert torch.equal(alone.codes(2, 25), codes[:2])
    codec = DacDecoderConfig(n_codebooks=4, codebook_size=256, latent_dim=64, channels=128, rates=(2, 4))
    audio = DacCodecDecoder(make_dac_weights(codec, seed=0), codec, device=gpu).from_indices(codes)
    assert audio.shape == (5, 1, 25 * codec.hop_length) and audio.isfinite().all()


def test_penalties_change_the_choice(gpu, example):
    """The same token twice in a row without a penalty for it; never with a large one."""
    config = example.TalkerConfig(codebooks=1, codebook_size=64)
    free = example.Talker(config, 1, gpu).codes(1, 40, repetition=1.0)[0, 0]
    held = example.Talker(config, 1, gpu).codes(1, 40, repetition=1e6)[0, 0]
    assert free.unique().numel() < 40
    assert held.unique().numel() == 40


@pytest.mark.parametrize("rows", [3, 70])
def test_captured_in_a_graph_and_on_a_side_stream(gpu, rows):
    """One capture of the four operators in a row, replayed on new inputs between eager work, and the
    same on a stream that is not the default one."""
    g = torch.Generator().manual_seed(rows)
    w = pack_block_fp8(torch.randn(512, 256, generator=g)).to(gpu)
    inv, _ = rotary_frequencies(64, device=gpu)
    x = torch.randn(rows, 256, generator=g).to(gpu)
    y = torch.randn(rows, 256, generator=g).to(torch.bfloat16).to(gpu)
    positions = torch.arange(rows, device=gpu)
    history = torch.randint(0, 512, (rows, 30), generator=g).to(gpu)
    lengths = torch.full((rows,), 30, device=gpu)
    penalty = torch.full((rows,), 1.5, device=gpu)

    def step():
        h, n = gated_residual_norm(x, y, post_norm=True, normed_dtype=torch.float8_e4m3fn)
        q = block_fp8_linear(n, w)
        r = apply_rotary(q.view(rows, 8, 64), None, positions, inv)
        z = block_fp8_linear(y, w, out_dtype=torch.float32)
        return h, q, r, adjust_logits(z, history=history, lengths=lengths, repetition=penalty)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            aside = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(aside, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(torch.randn(rows, 256, generator=g))
        y.copy_(torch.randn(rows, 256, generator=g))
        positions += k
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
