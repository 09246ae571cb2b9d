"""The gated residual norm against float64: both norms, every part alone and together, widths from
one channel to the largest, odd widths and strides, gates per channel, sequence and token, the 8-bit
output, rows of zeros and non-finite rows."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import BlockFp8Rows, gated_residual_norm

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
# A float32 sum over a row adds at most 32 terms in a thread, 6 levels in a wave and 16 waves: 54
# roundings; with the few of the formula itself, 64 of them bound each step.
STEP = 64 * 2.0 ** -24


def _norm64(v, err, norm, eps, weight, bias):
    """norm(v) in float64 and a bound on its float32 error, given one on v's."""
    mean = v.mean(1, keepdim=True) if norm == "layer" else torch.zeros_like(v[:, :1])
    d = v - mean
    rms = ((d * d).mean(1, keepdim=True) + eps).sqrt()
    # v's own error and the mean's, relative to the row's size, and the statistics' relative one
    err_d = err + (err.mean(1, keepdim=True) + STEP * v.abs().mean(1, keepdim=True)
                   if norm == "layer" else 0.0)
    rel = STEP + (err_d.pow(2).mean(1, keepdim=True)).sqrt() / rms
    n, en = d / rms, err_d / rms + d.abs() / rms * rel
    w = torch.ones_like(v[0]) if weight is None else weight.double()
    n, en = n * w, (en + STEP * n.abs()) * w.abs()
    if bias is not None:
        n, en = n + bias.double(), en + STEP * bias.double().abs()
    return n, en


def _reference(x, y, kw):
    norm, eps = kw.get("norm", "rms"), kw.get("eps", 1e-6)
    u, eu = y.double(), torch.zeros_like(y, dtype=torch.float64)
    if kw.get("post_norm"):
        u, eu = _norm64(u, eu, norm, eps, kw.get("post_weight"), kw.get("post_bias"))
    gate = kw.get("gate")
    if gate is not None:
        z = gate.double().reshape(-1, y.shape[1])
        act = kw.get("gate_activation", "none")
        g = {"none": z, "sigmoid": torch.sigmoid(z), "tanh": torch.tanh(z)}[act]
        g = g.repeat_interleave(y.shape[0] // z.shape[0], 0)
        eu = eu * g.abs() + STEP * (u * g).abs()
        u = u * g
    s = kw.get("scale", 1.0)
    s = torch.tensor(s, dtype=F32).double().item()
    h = x.double() + s * u
    eh = abs(s) * eu + STEP * (x.double().abs() + (s * u).abs())
    n, en = _norm64(h, eh, norm, eps, kw.get("pre_weight"), kw.get("pre_bias"))
    return h, eh, n, en


def _check(x, y, **kw):
    h, n = gated_residual_norm(x, y, **kw)
    rh, eh, rn, en = _reference(x, y, kw)
    assert h.dtype == x.dtype and n.dtype == kw.get("normed_dtype", y.dtype)
    assert ((h.double() - rh).abs() <= eh + HALF_ULP[h.dtype] * (rh.abs() + eh) + 2.0 ** -25).all()
    assert ((n.double() - rn).abs() <= en + HALF_ULP[n.dtype] * (rn.abs() + en) + 2.0 ** -25).all()


def _rand(gpu, g, *shape, dtype=F32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype).to(gpu)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("rows,c", [(1, 2), (5, 7), (3, 64), (9, 500), (2, 512), (5, 513), (4, 1000),
                                    (3, 1024), (7, 1025), (2, 2048), (3, 3000), (2, 4096),
                                    (3, 5001), (2, 8192), (2, 9000), (2, 16384), (2, 32768)])
def test_widths(gpu, norm, rows, c):
    g = torch.Generator().manual_seed(c)
    x, y = _rand(gpu, g, rows, c, std=2.0), _rand(gpu, g, rows, c, dtype=BF16)
    w = [_rand(gpu, g, c) for _ in range(4)]
    kw = {"post_norm": True, "post_weight": w[0], "pre_weight": w[1], "norm": norm, "eps": 1e-5}
    if norm == "layer":
        kw |= {"post_bias": w[2], "pre_bias": w[3]}
    _check(x, y, gate=_rand(gpu, g, c), scale=0.5, **kw)


@pytest.mark.parametrize("x_dtype,y_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F32, F16),
                                             (F16, F16)])
@pytest.mark.parametrize("normed", [F32, BF16, F16])
@pytest.mark.parametrize("c", [768, 333])
def test_types(gpu, x_dtype, y_dtype, normed, c):
    g = torch.Generator().manual_seed(c)
    x, y = _rand(gpu, g, 6, c, dtype=x_dtype), _rand(gpu, g, 6, c, dtype=y_dtype)
    for gate_dtype in (F32, BF16, F16):
        _check(x, y, gate=_rand(gpu, g, 6, c, dtype=gate_dtype), normed_dtype=normed)


@pytest.mark.parametrize("activation", ["none", "sigmoid", "tanh"])
@pytest.mark.parametrize("gates", [0, 1, 3, 12])
def test_gates(gpu, activation, gates):
    g = torch.Generator().manual_seed(gates)
    x, y = _rand(gpu, g, 12, 640, dtype=BF16), _rand(gpu, g, 12, 640, dtype=BF16)
    gate = _rand(gpu, g, gates, 640, dtype=BF16, std=3.0) if gates else _rand(gpu, g, 640, std=3.0)
    _check(x, y, gate=gate, gate_activation=activation, post_norm=True, scale=-1.5)
    if gates == 1:  # one gate expanded over the rows
        h, n = gated_residual_norm(x, y, gate=gate.expand(12, 640))
        h1, n1 = gated_residual_norm(x, y, gate=gate[0])
        assert torch.equal(h, h1) and torch.equal(n, n1)


def test_parts_left_out(gpu):
    g = torch.Generator().manual_seed(0)
    x, y = _rand(gpu, g, 4, 384), _rand(gpu, g, 4, 384)
    _check(x, y)
    _check(x, y, norm="layer")
    _check(x, y, post_norm=True)
    _check(x, y, pre_weight=_rand(gpu, g, 384))
    _check(x, y, norm="layer", pre_bias=_rand(gpu, g, 384), post_norm=True)


@pytest.mark.parametrize("c", [128, 100, 1000, 2064, 4096])
def test_eight_bit_output(gpu, c):
    """The 8-bit rows stand for the float32 rows: the same scale as their own largest value, up to
    the float32 statistics' last bits, and values within half an E4M3 step."""
    g = torch.Generator().manual_seed(c)
    x, y = _rand(gpu, g, 5, c), _rand(gpu, g, 5, c, dtype=BF16)
    w = _rand(gpu, g, c)
    x[1], y[1] = 0, 0
    h, q = gated_residual_norm(x, y, pre_weight=w, normed_dtype=torch.float8_e4m3fn)
    h32, n32 = gated_residual_norm(x, y, pre_weight=w, normed_dtype=F32)
    assert isinstance(q, BlockFp8Rows) and torch.equal(h, h32)
    assert q.values.shape == (5, -(-c // 16) * 16) and q.scale.shape == (5, -(-c // 128))
    assert (q.values.float()[:, c:] == 0).all() and (q.scale[1] == 1).all()
    pad = torch.nn.functional.pad(n32, (0, -c % 128)).view(5, -1, 128)
    amax = pad.abs().amax(2)
    assert torch.equal(q.scale[amax > 0], (amax / torch.full_like(amax, 448.0))[amax > 0])
    step = torch.maximum(n32.abs() * 2.0 ** -4,
                         q.scale.repeat_interleave(128, 1)[:, :c] * 2.0 ** -10)
    assert ((q.dequantized()[:, :c] - n32).abs() <= step * 1.001).all()


def test_strided_rows_and_in_place(gpu):
    g = torch.Generator().manual_seed(1)
    x = _rand(gpu, g, 9, 1100, dtype=BF16)[:, 3:1003]
    y = _rand(gpu, g, 9, 3000, dtype=BF16)[:, 1001:2001]
    gate = _rand(gpu, g, 9, 2000, dtype=BF16)[:, ::2][:, :1000].contiguous()
    want = gated_residual_norm(x.contiguous(), y.contiguous(), gate=gate)
    got = gated_residual_norm(x, y, gate=gate)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = gated_residual_norm(x, y, gate=gate, residual_out=x)
    assert got[0].data_ptr() == x.data_ptr() and torch.equal(x, want[0])
    assert torch.equal(got[1], want[1])


def test_many_rows_and_no_rows(gpu):
    g = torch.Generator().manual_seed(2)
    x, y = _rand(gpu, g, 3000, 256, dtype=BF16), _rand(gpu, g, 3000, 256, dtype=BF16)
    _check(x, y, post_norm=True)
    h, n = gated_residual_norm(x[:0], y[:0])
    assert h.shape == n.shape == (0, 256)


def test_zero_constant_and_non_finite_rows(gpu):
    g = torch.Generator().manual_seed(3)
    x, y = _rand(gpu, g, 6, 700), _rand(gpu, g, 6, 700)
    clean = gated_residual_norm(x, y, norm="layer", post_norm=True)
    x[0], y[0] = 0, 0
    y[1] = 5.0  # no variance: the layer norm leaves 0
    x[2, 3], y[3, 699] = float("nan"), float("inf")
    h, n = gated_residual_norm(x, y, norm="layer", post_norm=True)
    assert (h[0] == 0).all() and (n[0] == 0).all()
    assert torch.equal(h[1], x[1])
    assert n[2].isnan().all() and h[3].isnan().all()
    for got, want in zip((h, n), clean):
        assert torch.equal(got[4:], want[4:])


def test_refusals(gpu):
    x, y = torch.zeros(4, 64, device=gpu), torch.zeros(4, 64, device=gpu, dtype=BF16)
    w = torch.zeros(64, device=gpu)
    bad = [
        dict(norm="group"), dict(gate_activation="relu", gate=w), dict(gate_activation="tanh"),
        dict(pre_bias=w), dict(post_weight=w), dict(pre_weight=w[:63]), dict(pre_weight=w.half()),
        dict(gate=torch.zeros(3, 64, device=gpu)), dict(gate=torch.zeros(4, 63, device=gpu)),
        dict(gate=w.double()), dict(normed_dtype=torch.float64),
        dict(residual_out=torch.zeros(4, 64, device=gpu, dtype=BF16)),
    ]
    for kw in bad:
        with pytest.raises(ValueError):
            gated_residual_norm(x, y, **kw)
    with pytest.raises(ValueError):
        gated_residual_norm(x[:3], y)
    with pytest.raises(ValueError):
        gated_residual_norm(x.half(), y)
    with pytest.raises(ValueError):
        gated_residual_norm(x.t(), y.t())
    with pytest.raises(N.OmniCodecError):
        gated_residual_norm(x.cpu(), y.cpu())
    with pytest.raises(N.OmniCodecError) as refused:
        gated_residual_norm(torch.zeros(1, 32769, device=gpu), torch.zeros(1, 32769, device=gpu))
    assert refused.value.status == N.UNSUPPORTED
    with pytest.raises(N.OmniCodecError) as refused:
        gated_residual_norm(x, y, eps=-1.0)
    assert refused.value.status == N.INVALID_ARG
