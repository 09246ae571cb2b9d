"""Rope scalings as configurations write them: every key is honoured or refused, against each
definition written out for single pairs."""

from __future__ import annotations

import math

import pytest
import torch

from sglang_omni_amd.kernels import rotary_frequencies

YARN = {"rope_type": "yarn", "factor": 40.0, "original_max_position_embeddings": 4096}


def _yarn_by_hand(dim, base, factor, original, truncate, fast=32.0, slow=1.0):
    """Each pair on its own, from its number of turns in the original context."""
    ends = [dim * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base))
            for turns in (fast, slow)]
    if truncate:
        ends = [math.floor(ends[0]), math.ceil(ends[1])]
    low, high = max(ends[0], 0), min(ends[1], dim - 1)
    out = []
    for i in range(dim // 2):
        kept = base ** (-2 * i / dim)
        share = min(max((i - low) / (high - low), 0.0), 1.0)
        out.append(kept * (1 - share) + kept / factor * share)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("dim,base,extra,factor", [
    (64, 1e4, {}, 0.1 * math.log(40) + 1),
    (64, 1e4, {"mscale": 1.0, "mscale_all_dim": 1.0}, 1.0),
    (64, 1e4, {"mscale": 0.707, "mscale_all_dim": 0.707}, 1.0),
    (128, 1e6, {"mscale": 1.0, "mscale_all_dim": 0.5},
     (0.1 * math.log(40) + 1) / (0.05 * math.log(40) + 1)),
    (64, 1e4, {"mscale": 1.0, "mscale_all_dim": 0.0}, 0.1 * math.log(40) + 1),
    (64, 1e4, {"mscale": 0.707, "mscale_all_dim": 0.5, "attention_factor": 1.25}, 1.25),
    (64, 1.5e5, {"truncate": False}, 0.1 * math.log(40) + 1),
    (96, 1.5e5, {"truncate": False, "beta_fast": 24.0, "beta_slow": 2.0}, 0.1 * math.log(40) + 1),
    (64, 1.5e5, {"truncate": True, "beta_fast": 16, "beta_slow": None}, 0.1 * math.log(40) + 1),
])
def test_yarn(dim, base, extra, factor):
    got, got_factor = rotary_frequencies(dim, base, {**YARN, **extra})
    want = _yarn_by_hand(dim, base, 40.0, 4096, extra.get("truncate", True),
                         extra.get("beta_fast") or 32.0, extra.get("beta_slow") or 1.0)
    assert torch.allclose(got, want, rtol=1e-12, atol=0)
    assert got_factor == pytest.approx(factor, rel=1e-12)


def test_longrope():
    scaling = {"rope_type": "longrope", "long_factor": [1.0, 2.0, 3.0, 4.0],
               "short_factor": [1.0, 1.1, 1.2, 1.3], "original_max_position_embeddings": 4096}
    with pytest.raises(ValueError, match="factor"):  # the ratio of the contexts, not here to take
        rotary_frequencies(8, 1e4, scaling)
    plain, _ = rotary_frequencies(8, 1e4)
    got, factor = rotary_frequencies(8, 1e4, {**scaling, "factor": 32.0})
    assert factor == pytest.approx(math.sqrt(1 + math.log(32) / math.log(4096)), rel=1e-12)
    assert torch.allclose(got, plain / torch.tensor([1.0, 2.0, 3.0, 4.0], dtype=torch.float64))
    short, _ = rotary_frequencies(8, 1e4, {**scaling, "factor": 32.0, "short": True})
    assert torch.allclose(short, plain / torch.tensor([1.0, 1.1, 1.2, 1.3], dtype=torch.float64))
    del scaling["original_max_position_embeddings"]
    _, given = rotary_frequencies(8, 1e4, {**scaling, "attention_factor": 1.25})
    assert given == 1.25


def test_base_within_the_scaling():
    same, _ = rotary_frequencies(64, 5e5, {**YARN, "rope_theta": 500000})
    assert torch.equal(same, rotary_frequencies(64, 5e5, YARN)[0])
    with pytest.raises(ValueError, match="rope_theta"):
        rotary_frequencies(64, 1e4, {**YARN, "rope_theta": 5e5})


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default", "mrope_section": [16, 24, 24]},
    {"mrope_section": [16, 24, 24]},
    {"rope_type": "default", "factor": 2.0},
    {"rope_type": "linear"},
    {"rope_type": "linear", "factor": 2.0, "partial_rotary_factor": 0.5},
    {"rope_type": "linear", "type": "yarn", "factor": 2.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0},
    {"rope_type": "yarn", "original_max_position_embeddings": 4096},
    {"rope_type": "yarn", "factor": 4.0},
    {**YARN, "mscale": 0.707},
    {**YARN, "mscale_all_dim": 1.0},
    {**YARN, "mscale": 0.707, "mscale_all_dim": 0.0},
    {**YARN, "finetuned": True},
    {**YARN, "beta_fast": 1, "beta_slow": 32},
    {**YARN, "original_max_position_embeddings": 4},
    {**YARN, "original_max_position_embeddings": 1},
    {"rope_type": "longrope", "factor": 32.0, "long_factor": [1.0] * 32},
    {"rope_type": "longrope", "factor": 32.0, "original_max_position_embeddings": 4096},
    {"rope_type": "dynamic", "factor": 2.0},
])
def test_refused(scaling):
    with pytest.raises(ValueError):
        rotary_frequencies(64, 1e4, scaling)
