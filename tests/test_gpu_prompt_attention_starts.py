"""Packed prompts that do not begin at row 0: the rows in front of the first sequence, like those
behind the last one, are zero in an output made by the call and stay as they are in one that is given."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd.kernels import prompt_attention
from tests.test_gpu_prompt_attention import exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,before,heads,kv,dim", [
    ([100, 0, 30], 0, 4, 2, 64), ([], 0, 4, 2, 64), ([700, 650], 0, 64, 16, 128), ([3], 6000, 4, 2, 128),
    ([500], 15000, 32, 4, 64), ([1] * 200, 0, 2, 1, 64), ([90], 0, 2, 1, 256)])
@pytest.mark.parametrize("front,rest", [(1, 0), (37, 5), (300, 300)])
def test_rows_in_front_of_the_first_sequence(gpu, causal, lengths, before, heads, kv, dim, front, rest):
    g = torch.Generator().manual_seed(front + dim)
    total = sum(lengths)
    q = torch.randn(front + total + rest, heads, dim, generator=g).to(torch.bfloat16).to(gpu)
    key_lengths = [n + before for n in lengths]
    k, v = (torch.randn(front + sum(key_lengths) + rest, kv, dim, generator=g).to(torch.bfloat16).to(gpu)
            for _ in range(2))
    starts, key_starts = (torch.tensor([front, *n], device=gpu).cumsum(0) for n in (lengths, key_lengths))
    last = front + total
    used = torch.full_like(q, float("nan"))
    del used  # what memory an output finds
    got = prompt_attention(q, k, v, starts, key_starts=key_starts, causal=causal)
    assert (got[:front] == 0).all() and (got[last:] == 0).all()
    want, bound = exact(q[front:], k[front:], v[front:], lengths, key_lengths, causal, dim ** -0.5)
    assert ((got[front:last].double() - want[:total]).abs() <= bound[:total]).all()
    out = torch.full_like(q, 7.0)
    prompt_attention(q, k, v, starts, key_starts=key_starts, causal=causal, out=out)
    assert torch.equal(out[front:last], got[front:last])
    assert (out[:front] == 7).all() and (out[last:] == 7).all()
