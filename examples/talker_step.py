"""A small talker in 8-bit floating point, from its tokens to audio.

The codec decodes codes; this is the loop that makes them, on the same kernels: block-scaled 8-bit
linear layers, gated residual norms that hand the next linear layer its 8-bit rows, rotary positions
scaled for a long context, sliding-window attention over the slots' K / V rings, and logits adjusted
by repetition penalties, a bias and a mask that lets each step emit its own codebook only. The codes
of all streams then go through a DAC-style decoder.

Run on a GPU, with the library built:

    PYTHONPATH=sglang-omni_amd python examples/talker_step.py --streams 8 --frames 12

Weights are random; the audio is noise.
"""

from __future__ import annotations

import argparse
from dataclasses import dataclass

import torch

from sglang_omni_amd.kernels import (BlockFp8Rows, BlockFp8Weight, adjust_logits, apply_rotary,
                                     block_fp8_linear, gated_residual_norm, pack_block_fp8,
                                     rotary_frequencies)
from sglang_omni_amd.kernels.code2wav_front import silu_mul, window_attention
from sglang_omni_amd.models import DacCodecDecoder, DacDecoderConfig, make_dac_weights


@dataclass(frozen=True)
class TalkerConfig:
    codebooks: int = 4
    codebook_size: int = 256
    hidden: int = 512
    layers: int = 2
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    intermediate: int = 1024
    window: int = 72
    layer_scale: float = 0.5
    eps: float = 1e-5

    @property
    def vocab(self) -> int:
        return self.codebooks * self.codebook_size


@dataclass
class Layer:
    qkv: BlockFp8Weight
    o: BlockFp8Weight
    gate_up: BlockFp8Weight
    down: BlockFp8Weight
    norms: tuple[torch.Tensor, ...]  # before attention, after it, before the MLP, after it
    scales: tuple[torch.Tensor, torch.Tensor]  # of the attention's and the MLP's output, per channel


class Talker:
    """The weights, and for `slots` streams the K / V rings, positions and the last `history` tokens."""

    def __init__(self, config: TalkerConfig, slots: int, device: torch.device, seed: int = 0,
                 history: int = 4096):
        c = self.config = config
        g = torch.Generator().manual_seed(seed)

        def linear(n: int, k: int) -> BlockFp8Weight:
            return pack_block_fp8(torch.randn(n, k, generator=g) * k ** -0.5).to(device)

        def vector(mean: float) -> torch.Tensor:
            return (mean * (1 + 0.1 * torch.randn(c.hidden, generator=g))).to(device)

        kv = c.kv_heads * c.head_dim
        width = c.heads * c.head_dim
        self.embedding = torch.randn(c.vocab, c.hidden, generator=g).to(torch.bfloat16).to(device)
        self.layers = [Layer(linear(width + 2 * kv, c.hidden), linear(c.hidden, width),
                             linear(2 * c.intermediate, c.hidden), linear(c.hidden, c.intermediate),
                             tuple(vector(1.0) for _ in range(4)),
                             (vector(c.layer_scale), vector(c.layer_scale)))
                       for _ in range(c.layers)]
        self.final_norm = vector(1.0)
        self.head = linear(c.vocab, c.hidden)
        self.inv_freq, self.rotary_factor = rotary_frequencies(
            c.head_dim, 10000.0, {"rope_type": "yarn", "factor": 4.0,
                                  "original_max_position_embeddings": 2048}, device=device)
        self.rings = [[torch.zeros(slots * c.window, kv, dtype=torch.bfloat16, device=device)
                       for _ in range(2)] for _ in range(c.layers)]
        self.positions = torch.zeros(slots, dtype=torch.int64, device=device)
        self.history = torch.zeros(slots, history, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(slots, dtype=torch.int32, device=device)
        # mask q allows the tokens of codebook q
        token = torch.arange(c.vocab).view(-1, 32) // c.codebook_size
        bits = 1 << torch.arange(32, dtype=torch.int64)
        masks = torch.stack([((token == q) * bits).sum(1) for q in range(c.codebooks)])
        self.allowed = masks.to(torch.int32).to(device)

    def hidden_rows(self, tokens: torch.Tensor, slot_index: torch.Tensor) -> BlockFp8Rows:
        """One token of each stream through the layers: the head's 8-bit input rows."""
        c = self.config
        batch = tokens.shape[0]
        width, kv = c.heads * c.head_dim, c.kv_heads * c.head_dim
        positions = self.positions[slot_index]
        ring_rows = slot_index * c.window + positions % c.window
        x = self.embedding[tokens]
        h, rows = gated_residual_norm(torch.zeros_like(x, dtype=torch.float32), x, eps=c.eps,
                                      pre_weight=self.layers[0].norms[0],
                                      normed_dtype=torch.float8_e4m3fn)
        for n, (layer, (key_ring, value_ring)) in enumerate(zip(self.layers, self.rings)):
            qkv = block_fp8_linear(rows, layer.qkv)
            q = qkv[:, :width].view(batch, c.heads, c.head_dim)
            k = qkv[:, width:width + kv].view(batch, c.kv_heads, c.head_dim)
            apply_rotary(q, k, positions, self.inv_freq, factor=self.rotary_factor, q_out=q, k_out=k)
            key_ring[ring_rows] = qkv[:, width:width + kv]
            value_ring[ring_rows] = qkv[:, width + kv:]
            attended = torch.empty(batch, width, dtype=torch.bfloat16, device=qkv.device)
            window_attention(qkv, batch, c.heads, c.kv_heads, c.head_dim, c.window,
                             c.head_dim ** -0.5, attended, slot_index=slot_index,
                             positions=self.positions, cold=False, key_ring=key_ring,
                             value_ring=value_ring, ring_frames=c.window)
            y = block_fp8_linear(attended, layer.o)
            h, rows = gated_residual_norm(h, y, eps=c.eps, post_norm=True,
                                          post_weight=layer.norms[1], gate=layer.scales[0],
                                          pre_weight=layer.norms[2], residual_out=h,
                                          normed_dtype=torch.float8_e4m3fn)
            gate_up = block_fp8_linear(rows, layer.gate_up)
            mlp = torch.empty(batch, c.intermediate, dtype=torch.bfloat16, device=qkv.device)
            y = block_fp8_linear(silu_mul(gate_up, mlp), layer.down)
            following = self.layers[n + 1].norms[0] if n + 1 < c.layers else self.final_norm
            h, rows = gated_residual_norm(h, y, eps=c.eps, post_norm=True,
                                          post_weight=layer.norms[3], gate=layer.scales[1],
                                          pre_weight=following, residual_out=h,
                                          normed_dtype=torch.float8_e4m3fn)
        self.positions[slot_index] += 1
        return rows

    def step(self, tokens: torch.Tensor, slot_index: torch.Tensor, codebook: int,
             repetition: torch.Tensor, bias_tokens: torch.Tensor | None = None,
             bias_values: torch.Tensor | None = None) -> torch.Tensor:
        """The next token of each stream, of codebook `codebook`: the likeliest after the penalties."""
        rows = self.hidden_rows(tokens, slot_index)
        logits = block_fp8_linear(rows, self.head, out_dtype=torch.float32)
        adjust_logits(logits, history=self.history, lengths=self.lengths, slot_index=slot_index,
                      repetition=repetition, bias_tokens=bias_tokens, bias_values=bias_values,
                      allowed=self.allowed, allowed_index=torch.full_like(slot_index, codebook),
                      out=logits)
        nxt = logits.argmax(1)
        # the history is a ring: the penalties are those of a stream's last tokens
        at = self.lengths[slot_index].long() % self.history.shape[1]
        self.history[slot_index, at] = nxt.to(torch.int32)
        self.lengths[slot_index] += 1
        return nxt

    def codes(self, streams: int, frames: int, repetition: float = 1.3) -> torch.Tensor:
        """`frames` frames of codes [streams, codebooks, frames] for slots 0 .. streams - 1."""
        c, device = self.config, self.embedding.device
        slots = torch.arange(streams, device=device)
        penalty = torch.full((streams,), repetition, device=device)
        tokens = torch.arange(streams, device=device) % c.vocab
        out = torch.empty(streams, c.codebooks, frames, dtype=torch.int64, device=device)
        for t in range(frames):
            for q in range(c.codebooks):
                tokens = self.step(tokens, slots, q, penalty)
                out[:, q, t] = tokens - q * c.codebook_size
        return out


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n", 1)[0])
    parser.add_argument("--streams", type=int, default=8)
    parser.add_argument("--frames", type=int, default=12)
    args = parser.parse_args()
    device = torch.device("cuda", 0)
    config = TalkerConfig()
    talker = Talker(config, args.streams, device)
    codec = DacDecoderConfig(n_codebooks=config.codebooks, codebook_size=config.codebook_size,
                             latent_dim=64, channels=128, rates=(2, 4))
    decoder = DacCodecDecoder(make_dac_weights(codec, seed=0), codec, device=device)
    codes = talker.codes(args.streams, args.frames)
    audio = decoder.from_indices(codes)
    print(f"{args.streams} streams x {args.frames} frames of {config.codebooks} codes -> audio "
          f"{tuple(audio.shape)}, rms {audio.float().pow(2).mean().sqrt().item():.3f}")


if __name__ == "__main__":
    main()
