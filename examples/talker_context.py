"""A small talker that attends to its whole context: prompts of text into a paged key-value cache, then
one code after another, and the codes to audio.

The loop of talker_step.py attends to a window; this one keeps every key and value. A prompt's queries,
keys and values are normed and turned in one pass that also writes the cache, its attention runs over
the packed prompts (a later piece of a prompt reads what came before back from the cache), and each new
code attends to its stream's pages. The cache may hold 8 bits.

Run on a GPU, with the library built:

    PYTHONPATH=sglang-omni_amd python examples/talker_context.py --streams 8 --frames 12 --cache e4m3

Weights are random; the audio is noise.
"""

from __future__ import annotations

import argparse
from dataclasses import dataclass
from typing import Callable

import torch

from sglang_omni_amd.kernels import (BlockFp8Weight, PagedKvCache, adjust_logits, block_fp8_linear,
                                     gated_residual_norm, norm_rotary, pack_block_fp8, paged_attention,
                                     prompt_attention, read_kv_cache, rotary_frequencies)
from sglang_omni_amd.kernels.code2wav_front import silu_mul
from sglang_omni_amd.models import DacCodecDecoder, DacDecoderConfig, make_dac_weights

CACHES = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


@dataclass(frozen=True)
class ContextTalkerConfig:
    text_vocab: int = 512
    codebooks: int = 4
    codebook_size: int = 256
    hidden: int = 512
    layers: int = 2
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    intermediate: int = 1024
    page_size: int = 16
    eps: float = 1e-5

    @property
    def vocab(self) -> int:
        return self.text_vocab + self.codebooks * self.codebook_size


@dataclass
class Layer:
    qkv: BlockFp8Weight
    o: BlockFp8Weight
    gate_up: BlockFp8Weight
    down: BlockFp8Weight
    norms: tuple[torch.Tensor, torch.Tensor]  # before attention, before the MLP
    q_norm: torch.Tensor
    k_norm: torch.Tensor
    cache: PagedKvCache


class ContextTalker:
    """The weights, and a cache of `pages` pages a layer, handed out to streams as they grow."""

    def __init__(self, config: ContextTalkerConfig, streams: int, pages: int, device: torch.device,
                 seed: int = 0, cache_dtype: torch.dtype = torch.bfloat16):
        c = self.config = config
        g = torch.Generator().manual_seed(seed)

        def linear(n: int, k: int) -> BlockFp8Weight:
            return pack_block_fp8(torch.randn(n, k, generator=g) * k ** -0.5).to(device)

        def vector(n: int) -> torch.Tensor:
            return (1 + 0.1 * torch.randn(n, generator=g)).to(device)

        width, kv = c.heads * c.head_dim, c.kv_heads * c.head_dim
        self.embedding = torch.randn(c.vocab, c.hidden, generator=g).to(torch.bfloat16).to(device)
        self.layers = [Layer(linear(width + 2 * kv, c.hidden), linear(c.hidden, width),
                             linear(2 * c.intermediate, c.hidden), linear(c.hidden, c.intermediate),
                             (vector(c.hidden), vector(c.hidden)), vector(c.head_dim),
                             vector(c.head_dim),
                             PagedKvCache.allocate(pages, c.page_size, c.kv_heads, c.head_dim,
                                                   cache_dtype, device))
                       for _ in range(c.layers)]
        self.final_norm, self.head = vector(c.hidden), linear(c.vocab, c.hidden)
        self.inv_freq, _ = rotary_frequencies(c.head_dim, 10000.0, device=device)
        # the streams' pages and lengths, on the host, and the pages in the device's table
        self.free = list(range(pages))
        self.pages: list[list[int]] = [[] for _ in range(streams)]
        self.lengths = [0] * streams
        self.table = torch.zeros(streams, pages, dtype=torch.int32, device=device)
        token = torch.arange(-(-c.vocab // 32) * 32).view(-1, 32) - c.text_vocab
        bits = 1 << torch.arange(32, dtype=torch.int64)
        masks = [(((token >= 0) & (token // c.codebook_size == q)) * bits).sum(1)
                 for q in range(c.codebooks)]
        self.allowed = torch.stack(masks).to(torch.int32).to(device)

    def grow(self, streams: list[int], tokens: list[int]) -> list[int]:
        """Room for so many more tokens of each stream, of all of them or of none: their slots."""
        c = self.config
        if len(set(streams)) != len(streams) or min(tokens) < 1:
            raise ValueError("a call takes one token or more of each of its streams, each once")
        wanted = [-(-(self.lengths[s] + n) // c.page_size) - len(self.pages[s])
                  for s, n in zip(streams, tokens)]
        if sum(wanted) > len(self.free):
            raise RuntimeError("no free page")
        slots = []
        for s, n, more in zip(streams, tokens, wanted):
            for _ in range(more):
                self.pages[s].append(self.free.pop())
                self.table[s, len(self.pages[s]) - 1] = self.pages[s][-1]
            slots += self.slots(s, self.lengths[s], self.lengths[s] + n)
            self.lengths[s] += n
        return slots

    def slots(self, stream: int, start: int, end: int) -> list[int]:
        size = self.config.page_size
        return [self.pages[stream][t // size] * size + t % size for t in range(start, end)]

    def release(self, stream: int) -> None:
        self.free += self.pages[stream]
        self.pages[stream], self.lengths[stream] = [], 0

    def _layers(self, tokens: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                attend: Callable) -> torch.Tensor:
        """tokens [n] through the layers: the head's logits [n, vocab]."""
        c = self.config
        n, device = tokens.shape[0], tokens.device
        x = self.embedding[tokens]
        h, rows = gated_residual_norm(torch.zeros_like(x, dtype=torch.float32), x, eps=c.eps,
                                      pre_weight=self.layers[0].norms[0],
                                      normed_dtype=torch.float8_e4m3fn)
        for i, layer in enumerate(self.layers):
            qkv = block_fp8_linear(rows, layer.qkv).view(n, -1, c.head_dim)
            q, k, v = qkv.split([c.heads, c.kv_heads, c.kv_heads], 1)
            q, k = norm_rotary(q, k, positions, self.inv_freq, q_weight=layer.q_norm,
                               k_weight=layer.k_norm, eps=c.eps, v=v, cache=layer.cache, slots=slots)
            attended = attend(layer.cache, q, k, v)
            y = block_fp8_linear(attended.view(n, -1), layer.o)
            h, rows = gated_residual_norm(h, y, eps=c.eps, pre_weight=layer.norms[1], residual_out=h,
                                          normed_dtype=torch.float8_e4m3fn)
            mlp = torch.empty(n, c.intermediate, dtype=torch.bfloat16, device=device)
            y = block_fp8_linear(silu_mul(block_fp8_linear(rows, layer.gate_up), mlp), layer.down)
            following = self.layers[i + 1].norms[0] if i + 1 < c.layers else self.final_norm
            h, rows = gated_residual_norm(h, y, eps=c.eps, pre_weight=following, residual_out=h,
                                          normed_dtype=torch.float8_e4m3fn)
        return block_fp8_linear(rows, self.head, out_dtype=torch.float32)

    def prompt(self, tokens: list[list[int]], streams: list[int]) -> torch.Tensor:
        """The next tokens of each stream's prompt, one after the other in one packed pass: the logits
        after each stream's last one."""
        device = self.embedding.device
        before = [self.lengths[s] for s in streams]
        slots = self.grow(streams, [len(t) for t in tokens])
        ends = torch.tensor([len(t) for t in tokens]).cumsum(0)
        starts = torch.cat([ends.new_zeros(1), ends]).to(device)
        positions = torch.tensor([b + i for b, t in zip(before, tokens) for i in range(len(t))],
                                 device=device)
        if not any(before):
            def attend(cache, q, k, v):
                return prompt_attention(q, k, v, starts)
        else:  # the keys of the streams' earlier pieces are in the cache, and by now these ones too
            whole = torch.tensor([slot for s in streams for slot in self.slots(s, 0, self.lengths[s])],
                                 device=device)
            key_ends = torch.tensor([self.lengths[s] for s in streams]).cumsum(0)
            key_starts = torch.cat([key_ends.new_zeros(1), key_ends]).to(device)

            def attend(cache, q, k, v):
                return prompt_attention(q, *read_kv_cache(cache, whole, dtype=q.dtype), starts,
                                        key_starts=key_starts)
        flat = torch.tensor([t for row in tokens for t in row], device=device)
        logits = self._layers(flat, positions, torch.tensor(slots, device=device), attend)
        return logits[starts[1:] - 1]

    def step(self, tokens: torch.Tensor, streams: list[int]) -> torch.Tensor:
        """One more token of each stream: the logits after it."""
        device = self.embedding.device
        positions = torch.tensor([self.lengths[s] for s in streams], device=device)
        slots = torch.tensor(self.grow(streams, [1] * len(streams)), device=device)
        longest = max(self.lengths[s] for s in streams)
        table = self.table[streams]

        def attend(cache, q, k, v):
            return paged_attention(q, cache, table, positions + 1, max_length=longest)

        return self._layers(tokens, positions, slots, attend)

    def codes(self, prompts: list[list[int]], frames: int) -> torch.Tensor:
        """`frames` frames of codes [streams, codebooks, frames] after the prompts of streams 0 ..."""
        c, device = self.config, self.embedding.device
        streams = list(range(len(prompts)))
        logits = self.prompt(prompts, streams)
        out = torch.empty(len(prompts), c.codebooks, frames, dtype=torch.int64, device=device)
        for t in range(frames):
            for q in range(c.codebooks):
                if t or q:
                    logits = self.step(tokens, streams)
                book = torch.full((len(prompts),), q, device=device)
                adjust_logits(logits, allowed=self.allowed, allowed_index=book, out=logits)
                tokens = logits.argmax(1)
                out[:, q, t] = tokens - c.text_vocab - q * c.codebook_size
        return out


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n", 1)[0])
    parser.add_argument("--streams", type=int, default=8)
    parser.add_argument("--frames", type=int, default=12)
    parser.add_argument("--cache", choices=sorted(CACHES), default="bf16")
    args = parser.parse_args()
    device = torch.device("cuda", 0)
    config = ContextTalkerConfig()
    talker = ContextTalker(config, args.streams, 64 * args.streams, device,
                           cache_dtype=CACHES[args.cache])
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, config.text_vocab, (20 + 37 * s,), generator=g).tolist()
               for s in range(args.streams)]
    codes = talker.codes(prompts, args.frames)
    codec = DacDecoderConfig(n_codebooks=config.codebooks, codebook_size=config.codebook_size,
                             latent_dim=64, channels=128, rates=(2, 4))
    audio = DacCodecDecoder(make_dac_weights(codec, seed=0), codec, device=device).from_indices(codes)
    print(f"{args.streams} prompts of up to {max(map(len, prompts))} tokens, {args.frames} frames of "
          f"{config.codebooks} codes -> audio {tuple(audio.shape)}, rms "
          f"{audio.float().pow(2).mean().sqrt().item():.3f}")


if __name__ == "__main__":
    main()
