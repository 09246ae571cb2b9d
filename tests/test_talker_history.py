"""The talker example's token history past its capacity, on the CPU: it holds the last tokens, and
nothing is written outside it."""

from __future__ import annotations

import importlib.util
import sys
from pathlib import Path

import pytest
import torch

_SPEC = importlib.util.spec_from_file_location(
    "talker_step", Path(__file__).resolve().parents[1] / "examples" / "talker_step.py")


@pytest.fixture(scope="module")
def example():
    module = importlib.util.module_from_spec(_SPEC)
    sys.modules["talker_step"] = module
    _SPEC.loader.exec_module(module)
    return module


@pytest.mark.parametrize("steps", [3, 5, 6, 23])
def test_full_history_keeps_the_last_tokens(example, monkeypatch, steps):
    """`step` itself, its kernels replaced: logits that name a given token, and the adjustments
    recorded as the operator reads them."""
    capacity = 5
    config = example.TalkerConfig(codebooks=1, codebook_size=64, hidden=64, layers=1, heads=1,
                                  kv_heads=1, intermediate=64)
    talker = example.Talker(config, 3, torch.device("cpu"), history=capacity)
    made, seen = [], []

    def logits(rows, head, out_dtype):
        made.append([(7 * len(made) + 3 * s) % config.vocab for s in range(2)])
        return torch.nn.functional.one_hot(torch.tensor(made[-1]), config.vocab).float()

    def adjust(logits, *, history, lengths, slot_index, **_):
        held = lengths[slot_index].clamp(max=history.shape[1])
        seen.append([sorted(history[s, :n].tolist()) for s, n in zip(slot_index, held)])

    monkeypatch.setattr(talker, "hidden_rows", lambda tokens, slot_index: None)
    monkeypatch.setattr(example, "block_fp8_linear", logits)
    monkeypatch.setattr(example, "adjust_logits", adjust)
    slots = torch.tensor([2, 0])
    tokens = torch.zeros(2, dtype=torch.int64)
    for _ in range(steps):
        tokens = talker.step(tokens, slots, 0, torch.ones(2))
        assert tokens.tolist() == made[-1]
    for t, rows in enumerate(seen):
        for s, held in enumerate(rows):
            assert held == sorted(m[s] for m in made[max(0, t - capacity):t])
    assert talker.lengths.tolist() == [steps, 0, steps]
    assert (talker.history[1] == 0).all()
