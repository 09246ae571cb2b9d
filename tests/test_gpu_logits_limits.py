"""Limits of the logit adjustments: the largest history, and prompt lengths far below zero."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import adjust_logits


def test_counts_fit_their_words():
    """A token's count has 30 bits, so 2^30 tokens of history are refused. Without a GPU: the rows
    (2^31) are past what a launch takes, so 2^30 - 1 tokens are refused as unsupported instead."""
    fields = [name for name, _ in N.LogitsArgs._fields_]

    def status(capacity):
        values = dict.fromkeys(fields, 0)
        values |= {name: 4096 for name in ("logits", "out", "history", "lengths")}
        values |= {"dtype": N.DTYPE_F32, "out_dtype": N.DTYPE_F32, "tokens_dtype": N.DTYPE_I32,
                   "lengths_dtype": N.DTYPE_I32, "logits_stride": 64, "out_stride": 64, "vocab": 64,
                   "rows": 2**31, "slots": 2**31, "history_stride": capacity, "capacity": capacity}
        return N.load_library().omni_adjust_logits(N.pack_logits(*values.values()), None)

    assert status(2**30 - 1) == N.UNSUPPORTED
    assert status(2**30) == N.INVALID_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("first", [-1, -2**31, -2**32 + 3, -2**62 + 2])
def test_prompt_lengths_below_zero_are_none(gpu, first):
    logits = torch.randn(2, 100, generator=torch.Generator().manual_seed(1)).to(gpu)
    kw = {"history": torch.tensor([[5, 6, 5, 7], [1, 2, 3, 4]], device=gpu),
          "lengths": torch.tensor([4, 3], device=gpu),
          "frequency": torch.tensor([0.5, 0.25], device=gpu),
          "presence": torch.tensor([1.0, 2.0], device=gpu)}
    got = adjust_logits(logits, prompt_lengths=torch.tensor([first, first], device=gpu), **kw)
    assert torch.equal(got, adjust_logits(logits, **kw))
