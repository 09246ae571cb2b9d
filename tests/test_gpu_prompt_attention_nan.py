"""NaN in what a query of prompt attention sees is NaN in its output, whichever form takes the call and
whether its keys are split or not; a row whose scores are all -infinity is zero; neither reaches
another row."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import prompt_attention

pytestmark = pytest.mark.gpu

# queries, keys before them, heads, key heads; rows of a workgroup, keys in several pieces
FORMS = [(300, 0, 4, 2, 32, False), (3, 6000, 4, 2, 32, True), (1350, 0, 64, 16, 128, False),
         (500, 15000, 32, 4, 128, True)]


def inputs(gpu, form, dim, dtype, seed):
    queries, before, heads, kv, rows, split = form
    tile = N.ctypes.c_int()
    pieces = N.load_library().omni_prompt_plan(queries, queries + before, 1, heads, kv, dim, 1,
                                               N.ctypes.byref(tile))
    assert (tile.value, pieces > 1) == (rows, split)
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(queries, heads, dim, generator=g).to(dtype).to(gpu)
    k, v = (torch.randn(queries + before, kv, dim, generator=g).to(dtype).to(gpu) for _ in range(2))
    starts = torch.tensor([0, queries], device=gpu)
    return q, k, v, starts, torch.tensor([0, queries + before], device=gpu)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_a_query_of_nan(gpu, dtype, dim, form):
    q, k, v, starts, key_starts = inputs(gpu, form, dim, dtype, dim)
    clean = prompt_attention(q, k, v, starts, key_starts=key_starts)
    assert clean.isfinite().all()
    at, head = form[0] // 2, form[2] - 1
    q[at, head, 3] = float("nan")
    got = prompt_attention(q, k, v, starts, key_starts=key_starts)
    assert got[at, head].isnan().all()
    # the rows beside it share its wave's maxima: off by two roundings at most, of weights and result, on
    # either side; other key heads' rows keep their bits
    group = form[2] // form[3]
    off = (got[:, -group:].double() - clean[:, -group:].double()).abs()
    off[at, -1] = 0
    assert (off <= 4 * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -6) * v.float().abs().max().item()).all()
    assert torch.equal(got[:, :-group], clean[:, :-group])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_keys_of_nan(gpu, dim, form):
    """The first half of one head's keys, whole pieces of a split row: every query that sees one is NaN, and
    no query of another head is."""
    q, k, v, starts, key_starts = inputs(gpu, form, dim, torch.bfloat16, dim + 1)
    clean = prompt_attention(q, k, v, starts, key_starts=key_starts)
    group = form[2] // form[3]
    k[:k.shape[0] // 2, 1] = float("nan")
    got = prompt_attention(q, k, v, starts, key_starts=key_starts)
    mine = torch.arange(form[2], device=gpu) // group == 1
    assert got[:, mine].isnan().all()
    assert torch.equal(got[:, ~mine], clean[:, ~mine])


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("value", [1.0, float("inf"), float("nan")])
def test_scores_of_minus_infinity(gpu, dim, form, value):
    """All of a row's scores -infinity: zero, whatever the values are; the other rows are what they were."""
    q, k, v, starts, key_starts = inputs(gpu, form, dim, torch.bfloat16, dim + 2)
    q = q.abs() + 0.5
    at = form[0] // 2
    q[:, :, 5] = 0
    clean = prompt_attention(q, k, v, starts, key_starts=key_starts)
    q[at, :, 5] = 1
    k[..., 5] = -3e38  # the query's product with it and the rest of the score: -infinity in float32
    q[at] *= 2 ** 4
    clean_values = v.float().abs().max().item()
    v[..., 9] = value
    got = prompt_attention(q, k, v, starts, key_starts=key_starts)
    assert (got[at] == 0).all()
    # the rows beside it: as beside a NaN
    off = (got.double() - clean.double()).abs()
    off[at], off[..., 9] = 0, 0
    assert (off <= 2.0 ** -6 * (1 + 2.0 ** -6) * clean_values).all()
