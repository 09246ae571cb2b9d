"""Rotary positions against float64: both layouts, part of the head, every head width's vector
split, long positions, strides, in place, the transposed form as the gradient, and the scaled
frequencies' definitions (the frequencies themselves run without a GPU)."""

from __future__ import annotations

import math

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import apply_rotary, rotary_frequencies

HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def _turned64(t, positions, inv_freq, layout, factor, sign=1.0):
    angle = positions.double()[:, None] * inv_freq
    c, s = angle.cos()[:, None] * factor, sign * angle.sin()[:, None] * factor
    pairs = inv_freq.shape[0]
    v = t.double().clone()
    i = torch.arange(pairs, device=t.device)
    a_at, b_at = (i, i + pairs) if layout == "half" else (2 * i, 2 * i + 1)
    a, b = v[..., a_at], v[..., b_at]
    size = torch.zeros_like(v)
    size[..., a_at] = size[..., b_at] = (a.abs() + b.abs()) * factor
    v[..., a_at], v[..., b_at] = a * c - b * s, b * c + a * s
    return v, size


def _check(got, t, positions, inv_freq, layout, factor, sign=1.0):
    """sine and cosine within 2^-22 (their series, the reduced angle and the factor), two products
    and a sum, then one rounding to the type."""
    want, size = _turned64(t, positions, inv_freq, layout, factor, sign)
    bound = 2.0 ** -21 * size + HALF_ULP[t.dtype] * want.abs() + 2.0 ** -25
    assert got.dtype == t.dtype
    assert ((got.double() - want).abs() <= bound).all()
    rest = 2 * inv_freq.shape[0]
    assert torch.equal(got[..., rest:], t[..., rest:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary_dim", [(64, 64), (128, 128), (128, 64), (80, 40), (96, 32),
                                            (256, 256), (70, 70), (66, 2), (24, 12), (5, 4),
                                            (72, 36)])
def test_heads(gpu, dtype, layout, dim, rotary_dim):
    g = torch.Generator().manual_seed(dim + rotary_dim)
    inv, factor = rotary_frequencies(rotary_dim, 1e4, device=gpu)
    for tokens, heads, kv in ((1, 1, 1), (1, 16, 8), (7, 3, 2), (130, 5, 1)):
        qkv = torch.randn(tokens, (heads + 2 * kv) * dim + 3, generator=g).to(dtype).to(gpu)
        q = qkv[:, 1:1 + heads * dim].unflatten(1, (heads, dim))  # a view off the 16-byte grid
        k = qkv[:, 1 + heads * dim:1 + (heads + kv) * dim].unflatten(1, (kv, dim))
        positions = torch.randint(0, 200000, (tokens,), generator=g).to(gpu)
        qo, ko = apply_rotary(q, k, positions, inv, layout=layout, factor=1.25)
        _check(qo, q, positions, inv, layout, 1.25)
        _check(ko, k, positions, inv, layout, 1.25)
        assert torch.equal(apply_rotary(q, None, positions.int(), inv, layout=layout, factor=1.25), qo)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions_far_out_and_negative(gpu, layout):
    inv, _ = rotary_frequencies(128, 1e6, device=gpu)
    q = torch.randn(9, 2, 128, generator=torch.Generator().manual_seed(0)).to(gpu)
    positions = torch.tensor([0, 1, -1, -77777, 131071, 1000003, 2**31 - 1, 2**31 + 5, 16777217],
                             device=gpu)
    # float64 angles: 2^31 radians carry 2^-22 of rounding on both sides
    got = apply_rotary(q, None, positions, inv, layout=layout)
    _check(got, q, positions, inv, layout, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_in_place_and_strided_outputs(gpu, layout):
    g = torch.Generator().manual_seed(4)
    inv, _ = rotary_frequencies(48, device=gpu)
    qkv = torch.randn(33, 6 * 64, generator=g).to(torch.bfloat16).to(gpu)
    q, k = qkv[:, :256].view(33, 4, 64), qkv[:, 256:].view(33, 2, 64)
    positions = torch.arange(66, device=gpu)[::2]
    want = apply_rotary(q, k, positions, inv, layout=layout)
    buffer = torch.full((2, 4, 33, 64), float("nan"), dtype=torch.bfloat16, device=gpu)
    out = (buffer[0].transpose(0, 1), buffer[1, :2].transpose(0, 1))  # heads outside tokens
    got = apply_rotary(q, k, positions, inv, layout=layout, q_out=out[0], k_out=out[1])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert buffer[1, 2:].isnan().all()
    apply_rotary(q, k, positions, inv, layout=layout, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_transposed_is_the_gradient(gpu, layout):
    """Against the formula in float64, and against central differences of the forward form: it is
    linear, so a difference's only error is float32 rounding (2^-24 of the values around it, over
    the step)."""
    g = torch.Generator().manual_seed(6)
    inv, _ = rotary_frequencies(12, device=gpu)
    x, grad = (torch.randn(3, 2, 16, generator=g).to(gpu) for _ in range(2))
    positions = torch.tensor([3, 900, 77], device=gpu)
    got = apply_rotary(grad, None, positions, inv, layout=layout, factor=1.5, transposed=True)
    _check(got, grad, positions, inv, layout, 1.5, sign=-1.0)
    for at in ((0, 0, 0), (1, 1, 5), (2, 0, 7), (2, 1, 15)):
        plus, minus = x.clone(), x.clone()
        plus[at] += 1.0
        minus[at] -= 1.0
        f = [apply_rotary(v, None, positions, inv, layout=layout, factor=1.5).double()
             for v in (plus, minus)]
        slope = ((f[0] - f[1]) * grad.double()).sum() / (plus[at].double() - minus[at].double())
        assert abs(slope.item() - got[at].item()) <= 1e-4


@pytest.mark.gpu
def test_no_tokens_and_refusals(gpu):
    inv, _ = rotary_frequencies(32, device=gpu)
    q = torch.zeros(5, 2, 64, device=gpu)
    positions = torch.arange(5, device=gpu)
    assert apply_rotary(q[:0], None, positions[:0], inv).shape == (0, 2, 64)
    bad = [
        (q.double(), None, positions, inv, {}), (q[0], None, positions, inv, {}),
        (q.transpose(1, 2), None, positions, inv, {}), (q, None, positions[:4], inv, {}),
        (q, None, positions.float(), inv, {}), (q, None, positions, inv.float(), {}),
        (q[..., :30], None, positions, inv, {}), (q, q[:4], positions, inv, {}),
        (q, q.half(), positions, inv, {}), (q, None, positions, inv, {"layout": "neox"}),
        (q, None, positions, inv, {"k_out": q}), (q, None, positions, inv, {"q_out": q[:4]}),
        (q, None, positions, inv[:0], {}),
    ]
    for a, b, c, d, kw in bad:
        with pytest.raises(ValueError):
            apply_rotary(a, b, c, d, **kw)
    with pytest.raises(N.OmniCodecError):
        apply_rotary(q.cpu(), None, positions, inv)


def test_frequencies():
    inv, factor = rotary_frequencies(8, 10000.0)
    assert factor == 1.0 and inv.dtype == torch.float64
    assert torch.allclose(inv, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    linear, _ = rotary_frequencies(8, scaling={"rope_type": "linear", "factor": 4.0})
    assert torch.equal(linear, inv / 4)
    rope = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
            "original_max_position_embeddings": 1024}
    scaled, factor = rotary_frequencies(64, 500000.0, rope)
    plain, _ = rotary_frequencies(64, 500000.0)
    for p, s in zip(plain.tolist(), scaled.tolist()):
        wavelength = 2 * math.pi / p
        if wavelength < 1024 / 4.0:
            want = p
        elif wavelength > 1024 / 1.0:
            want = p / 8.0
        else:
            smooth = (1024 / wavelength - 1.0) / (4.0 - 1.0)
            want = (1 - smooth) * p / 8.0 + smooth * p
        assert s == pytest.approx(want, rel=1e-12)
    yarn, factor = rotary_frequencies(64, 10000.0, {"type": "yarn", "factor": 16.0,
                                                    "original_max_position_embeddings": 2048})
    plain, _ = rotary_frequencies(64, 10000.0)
    assert factor == pytest.approx(0.1 * math.log(16.0) + 1)
    turns = 2048 * plain / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], plain[turns > 40])
    assert torch.allclose(yarn[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-14)
    assert ((yarn <= plain) & (yarn >= plain / 16)).all()
    long = [1.0 + i for i in range(4)]
    got, factor = rotary_frequencies(8, scaling={
        "rope_type": "longrope", "factor": 32.0, "long_factor": long, "short_factor": [1.0] * 4,
        "original_max_position_embeddings": 4096})
    assert torch.allclose(got, inv / torch.tensor(long, dtype=torch.float64))
    assert factor == pytest.approx(math.sqrt(1 + math.log(32) / math.log(4096)))


def test_frequencies_refuse():
    for kw in ({"rotary_dim": 7}, {"rotary_dim": 0}, {"rotary_dim": 8, "base": 1.0},
               {"rotary_dim": 8, "scaling": {"rope_type": "wave"}},
               {"rotary_dim": 8, "scaling": {"rope_type": "linear", "factor": 0.5}},
               {"rotary_dim": 8, "scaling": {"rope_type": "longrope", "long_factor": [1.0],
                                             "original_max_position_embeddings": 64}}):
        with pytest.raises(ValueError):
            rotary_frequencies(**kw)
