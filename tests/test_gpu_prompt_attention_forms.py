"""Prompt attention in each of its forms (workgroups of 32 and of 128 rows, the keys of a row in one
piece and in several) where they can go wrong: infinities and NaN beside what a query sees, scores of
hundreds and maxima that grow and fall along the keys, capture in a graph."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import prompt_attention
from tests.test_gpu_prompt_attention import exact

pytestmark = pytest.mark.gpu

# queries, keys before them, heads, key heads; rows of a workgroup, keys in several pieces
FORMS = [(300, 0, 4, 2, 32, False), (70, 6000, 4, 2, 32, True), (1350, 0, 64, 16, 128, False),
         (500, 15000, 32, 4, 128, True)]


def inputs(gpu, form, dim, dtype, seed, std=1.0):
    queries, before, heads, kv, rows, split = form
    tile = N.ctypes.c_int()
    pieces = N.load_library().omni_prompt_plan(queries, queries + before, 1, heads, kv, dim, 1,
                                               N.ctypes.byref(tile))
    assert (tile.value, pieces > 1) == (rows, split)
    g = torch.Generator().manual_seed(seed)
    q = (std * torch.randn(queries, heads, dim, generator=g)).to(dtype).to(gpu)
    k, v = (torch.randn(queries + before, kv, dim, generator=g).to(dtype).to(gpu) for _ in range(2))
    starts = torch.tensor([0, queries], device=gpu)
    return q, k, v, starts, torch.tensor([0, queries + before], device=gpu)


def within(got, q, k, v, causal=True, scale=None, dims=slice(None)):
    """got's first and last group of heads against float64."""
    group = q.shape[1] // k.shape[1]
    for heads, kv_head in ((slice(0, group), slice(0, 1)), (slice(-group, None), slice(-1, None))):
        want, bound = exact(q[:, heads], k[:, kv_head], v[:, kv_head], [q.shape[0]], [k.shape[0]], causal,
                            q.shape[2] ** -0.5 if scale is None else scale)
        off = (got[:, heads].double() - want).abs()
        assert (off[..., dims] <= bound[..., dims]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_what_a_query_does_not_see_does_not_reach_it(gpu, dtype, bad, dim, form):
    queries, before, heads, kv = form[:4]
    q, k, v, starts, key_starts = inputs(gpu, form, dim, dtype, dim)
    group = heads // kv
    clean = prompt_attention(q, k, v, starts, key_starts=key_starts)
    for at in (1, 15, 32, 63, 64, queries // 2 + 1, queries - 1):
        for spoil_key in (False, True):
            k2, v2 = k.clone(), v.clone()
            v2[before + at, 0, 3] = bad
            if spoil_key:
                k2[before + at, 0] = bad
            got = prompt_attention(q, k2, v2, starts, key_starts=key_starts)
            assert torch.equal(got[:, group:], clean[:, group:])
            mine, keys = got[:, :group], (k2[:, :1], v2[:, :1])
            assert mine[:at].isfinite().all()
            want, bound = exact(q[:at, :group], *(t[:before + at] for t in keys), [at], [before + at], True,
                                dim ** -0.5)
            assert ((mine[:at].double() - want).abs() <= bound).all()
            if not spoil_key:
                assert not mine[at:, :, 3].isfinite().any()
                others = [d for d in range(dim) if d != 3]
                want, bound = exact(q[at:, :group], *keys, [queries - at], [before + queries], True, dim ** -0.5)
                assert ((mine[at:].double() - want).abs()[..., others] <= bound[..., others]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("std", [0.0, 0.01, 10.0, 40.0])
@pytest.mark.parametrize("form", FORMS)
def test_large_and_small_scores(gpu, dtype, dim, std, form):
    q, k, v, starts, key_starts = inputs(gpu, form, dim, dtype, dim + 1, std)
    ramp = torch.linspace(0, 4, k.shape[0], device=gpu)[:, None, None]
    for keys in (k, (k * ramp).to(dtype), (k * ramp.flip(0)).to(dtype)):
        within(prompt_attention(q, keys, v, starts, key_starts=key_starts), q, keys, v)
    got = prompt_attention(q, k, v, starts, key_starts=key_starts, scale=0.5, causal=False)
    within(got, q, k, v, False, 0.5)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("form", FORMS)
def test_captured_in_a_graph(gpu, dim, form):
    """Captured once, replayed on other inputs between eager work."""
    q, k, v, starts, key_starts = inputs(gpu, form, dim, torch.bfloat16, dim + 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        prompt_attention(q, k, v, starts, key_starts=key_starts)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = prompt_attention(q, k, v, starts, key_starts=key_starts)
    for _ in range(4):
        for t in (q, k, v):
            t.copy_(torch.randn_like(t))
        want = prompt_attention(q, k, v, starts, key_starts=key_starts)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
