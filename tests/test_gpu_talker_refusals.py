"""What the context talker of the examples refuses, and that a refused call leaves its streams as they
were: pieces without tokens, a stream twice in one call, more tokens than there are pages."""

from __future__ import annotations

import pytest
import torch

from tests.test_gpu_talker_context import example  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_refused_calls_leave_the_streams_as_they_were(gpu, example):  # noqa: F811
    config = example.ContextTalkerConfig()
    talker, other = (example.ContextTalker(config, 3, 8, gpu) for _ in range(2))
    first, following = [[1, 2, 3], [4] * 40], torch.tensor([7, 8], device=gpu)
    assert torch.equal(talker.prompt(first, [0, 1]), other.prompt(first, [0, 1]))

    def state():
        return talker.lengths[:], [p[:] for p in talker.pages], talker.free[:], talker.table.tolist()

    before = state()
    for tokens, streams in (([[5], []], [0, 1]), ([[], []], [0, 2]), ([[5], [6]], [1, 1])):
        with pytest.raises(ValueError):
            talker.prompt(tokens, streams)
    with pytest.raises(ValueError):
        talker.step(following, [1, 1])
    with pytest.raises(RuntimeError):  # room for the first stream's, not for the second's
        talker.prompt([[5] * 20, [6] * 90], [0, 1])
    assert state() == before
    assert torch.equal(talker.step(following, [0, 1]), other.step(following, [0, 1]))
