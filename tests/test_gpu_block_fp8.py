"""8-bit block-scaled linear layers and their row quantizer against float64, over row counts from one
to many tiles, odd columns, features that end inside a block, strides, and non-finite rows."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import (BlockFp8Rows, BlockFp8Weight, block_fp8_linear,
                                     block_fp8_weight, pack_block_fp8, quantize_block_rows)

pytestmark = pytest.mark.gpu

HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def _expanded(scale, per_row, rows, cols):
    return (scale.double().repeat_interleave(per_row, 0)[:rows]
            .repeat_interleave(128, 1)[:, :cols])


def _reference(x: BlockFp8Rows, w: BlockFp8Weight):
    """The product in float64, and per output the sum of the magnitudes of its terms."""
    a = x.values.double() * _expanded(x.scale, 1, *x.values.shape)
    b = w.weight.double() * _expanded(w.scale, 128, *w.weight.shape)
    y, size = a @ b.T, a.abs() @ b.abs().T
    if w.bias is not None:
        y, size = y + w.bias.double(), size + w.bias.double().abs()
    return y, size


def _check(y, x, w):
    """float32 sums of k products and k / 128 scaled blocks, each step within 2^-23 (rounded or cut)
    of the terms' magnitudes, then one rounding to the output's type."""
    want, size = _reference(x, w)
    k = x.values.shape[1]
    bound = (k + 8) * 2.0 ** -23 * size + HALF_ULP[y.dtype] * want.abs() + 2.0 ** -25
    assert ((y.double() - want).abs() <= bound).all()


def _operands(gpu, rows, k, n, seed, bias=False):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, k, generator=g) * torch.exp(torch.randn(k, generator=g))).to(gpu)
    w = torch.randn(n, k, generator=g).to(gpu) / k ** 0.5
    b = torch.randn(n, generator=g).to(gpu) if bias else None
    return x, pack_block_fp8(w, b)


def _quantized64(x):
    """The quantizer's definition group by group, its two quotients and the product in float32."""
    rows, k = x.shape
    kp, groups = -(-k // 16) * 16, -(-k // 128)
    q = torch.zeros(rows, kp, dtype=torch.float8_e4m3fn, device=x.device)
    s = torch.empty(rows, groups, device=x.device)
    for g in range(groups):
        part = x[:, g * 128:(g + 1) * 128].float()
        amax = part.abs().amax(1, keepdim=True)
        tiny, most = amax < 2.0 ** -100, torch.full_like(amax, 448.0)
        unit = torch.where(tiny, torch.ones_like(amax), most / amax)
        q[:, g * 128:g * 128 + part.shape[1]] = (part * unit).to(torch.float8_e4m3fn)
        s[:, g] = torch.where(tiny, torch.ones_like(amax), amax / most)[:, 0]
    return q, s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 15), (2, 128), (5, 129), (7, 1040), (300, 4096),
                                    (1, 8200), (33, 1000)])
def test_quantized_rows(gpu, dtype, rows, k):
    g = torch.Generator().manual_seed(rows * k)
    x = (torch.randn(rows, k + 3, generator=g) * 3).to(dtype).to(gpu)[:, 1:k + 1]  # strided, odd start
    x[0, k // 2] = 0
    if rows > 2:
        x[2] = 0
        x[1, :] *= 2.0 ** -20 if dtype == torch.float16 else 2.0 ** -99
    got = quantize_block_rows(x)
    q, s = _quantized64(x)
    assert got.values.shape == q.shape and torch.equal(got.scale, s)
    assert torch.equal(got.values.view(torch.uint8) & 0x7f, q.view(torch.uint8) & 0x7f)
    assert torch.equal(got.values.float(), q.float())


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,k,n", [
    (1, 16, 1), (1, 128, 16), (1, 1024, 2048), (2, 4096, 130), (7, 144, 33), (15, 640, 257),
    (16, 1024, 128), (17, 256, 1000), (31, 2048, 64), (33, 512, 515), (64, 1024, 1024),
    (65, 1040, 127), (128, 384, 512), (200, 896, 1536), (257, 1024, 2049), (513, 8192, 384)])
def test_linear(gpu, rows, k, n, out):
    x, w = _operands(gpu, rows, k, n, rows + k + n, bias=n % 2 == 1)
    q = quantize_block_rows(x)
    _check(block_fp8_linear(q, w, out_dtype=out), q, w)


@pytest.mark.parametrize("rows,k,n", [(300, 272, 4100), (530, 400, 4097), (2100, 272, 4100), (4099, 144, 3075),
                                      (700, 2064, 1300)])
def test_larger_tiles(gpu, rows, k, n):
    """Sizes that the tiles of 64 x 128, 128 x 128 and 256 x 256 take, ragged in every direction:
    float32 against float64, and bf16, whose products the 8-bit instruction cuts, against the bits of
    the small tiles on 40 rows at a time (every tile adds an element's blocks in one order)."""
    x, w = _operands(gpu, rows, k, n, rows, bias=True)
    q = quantize_block_rows(x)
    _check(block_fp8_linear(q, w, out_dtype=torch.float32), q, w)
    whole = block_fp8_linear(q, w)
    for at in (0, rows // 2, rows - 40):
        part = BlockFp8Rows(q.values[at:at + 40], q.scale[at:at + 40])
        assert torch.equal(block_fp8_linear(part, w), whole[at:at + 40])


@pytest.mark.parametrize("rows", [1, 16, 64, 200])
def test_operands_over_all_binades(gpu, rows):
    """Any E4M3 bit patterns. float32 output keeps the float32 bound. bf16 output may lose what the
    8-bit matrix instruction cuts: of 8 products added together each is cut below 2^-13 of the
    largest one's power of two, so 8 of them lose at most 7 * 2^-13 of the largest, whichever 8 of
    the block's 128 those are."""
    k, n = 384, 160
    g = torch.Generator().manual_seed(rows)

    def bits(r):
        b = torch.randint(0, 256, (r, k), generator=g).to(torch.uint8)
        b[(b & 0x7f) == 0x7f] = 0x11  # no NaN
        return b.to(gpu).view(torch.float8_e4m3fn)

    x = BlockFp8Rows(bits(rows), torch.rand(rows, 3, generator=g).to(gpu) + 0.1)
    w = BlockFp8Weight(bits(n), torch.rand(2, 3, generator=g).to(gpu) + 0.1)
    _check(block_fp8_linear(x, w, out_dtype=torch.float32), x, w)
    y = block_fp8_linear(x, w)
    want, size = _reference(x, w)
    a = (x.values.double() * _expanded(x.scale, 1, rows, k)).cpu()
    b = (w.weight.double() * _expanded(w.scale, 128, n, k)).cpu()
    cut = torch.zeros(rows, n, dtype=torch.float64)
    for block in range(3):
        p = (a[:, None, block * 128:(block + 1) * 128] * b[None, :, block * 128:(block + 1) * 128]).abs()
        cut += p.topk(16, dim=2).values.sum(2) * 7 * 2.0 ** -13  # 16 groups of 8, the worst grouping
    bound = cut.to(gpu) + (k + 8) * 2.0 ** -23 * size + HALF_ULP[y.dtype] * (want.abs() + cut.to(gpu))
    assert ((y.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("rows", [1, 4, 16, 40, 96, 300])
def test_float_rows_are_quantized_first(gpu, rows):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x, w = _operands(gpu, rows, 1040, 520, rows)
        x = x.to(dtype)
        q = quantize_block_rows(x)
        y = block_fp8_linear(x, w, out_dtype=torch.float32)
        _check(y, q, w)
        strided = torch.zeros(rows, 1100, dtype=dtype, device=gpu)[:, 5:1045].copy_(x)
        assert torch.equal(block_fp8_linear(strided, w, out_dtype=torch.float32), y)


def test_rows_do_not_depend_on_their_batch(gpu):
    """The same bits for a row whatever rows are batched with it, within each way of computing it:
    single tokens next to each other, and a prefill cut anywhere."""
    x, w = _operands(gpu, 700, 1536, 640, 5)
    q = quantize_block_rows(x)
    whole = block_fp8_linear(q, w)
    for rows in (700, 699, 640, 513):
        part = block_fp8_linear(BlockFp8Rows(q.values[:rows], q.scale[:rows]), w)
        assert torch.equal(part, whole[:rows])


def test_strided_operands_and_a_given_output(gpu):
    x, w = _operands(gpu, 70, 512, 300, 9, bias=True)
    q = quantize_block_rows(x)
    values = torch.zeros(70, 1024, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)[:, 256:768]
    values.view(torch.uint8).copy_(q.values.view(torch.uint8))
    scale = q.scale.t().contiguous().t()  # block-major
    weight = torch.zeros(300, 640, dtype=torch.uint8, device=gpu).view(torch.float8_e4m3fn)[:, :512]
    weight.view(torch.uint8).copy_(w.weight.view(torch.uint8))
    want = block_fp8_linear(q, w)
    buffer = torch.full((71, 307), float("nan"), dtype=torch.bfloat16, device=gpu)
    got = block_fp8_linear(BlockFp8Rows(values, scale), BlockFp8Weight(weight, w.scale, w.bias),
                           buffer[:70, 3:303])
    assert torch.equal(got, want)
    assert buffer[70].isnan().all() and buffer[:, :3].isnan().all() and buffer[:, 303:].isnan().all()


def test_bytes_past_the_features_are_not_read(gpu):
    """NaN bytes past k in the rows of both operands and past the last row leave no trace."""
    for rows in (3, 40, 300):
        k, n = 400, 72
        x, w = _operands(gpu, rows, k, n, rows)
        q = quantize_block_rows(x)
        pad = torch.full((rows + 40, 512), 0x7f, dtype=torch.uint8, device=gpu)
        pad[:rows, :k] = q.values.view(torch.uint8)
        wpad = torch.full((n + 40, 512), 0x7f, dtype=torch.uint8, device=gpu)
        wpad[:n, :k] = w.weight.view(torch.uint8)
        got = block_fp8_linear(
            BlockFp8Rows(pad.view(torch.float8_e4m3fn)[:rows, :k], q.scale),
            BlockFp8Weight(wpad.view(torch.float8_e4m3fn)[:n, :k], w.scale))
        assert torch.equal(got, block_fp8_linear(q, w))


def test_non_finite_rows_stay_their_own(gpu):
    for rows in (8, 80, 300):
        x, w = _operands(gpu, rows, 512, 192, rows)
        x = x.to(torch.bfloat16)
        clean = block_fp8_linear(x, w)
        x[3, 200] = float("nan")
        x[5, 7] = float("inf")
        got = block_fp8_linear(x, w)
        assert got[3].isnan().all() and got[5].isnan().all()
        keep = [r for r in range(rows) if r not in (3, 5)]
        assert torch.equal(got[keep], clean[keep])


def test_no_rows(gpu):
    _, w = _operands(gpu, 1, 256, 96, 0)
    x = torch.empty(0, 256, dtype=torch.bfloat16, device=gpu)
    assert block_fp8_linear(x, w).shape == (0, 96)
    assert quantize_block_rows(x).values.shape == (0, 256)


def test_packed_and_checkpoint_weights(gpu):
    g = torch.Generator().manual_seed(3)
    w = torch.randn(200, 300, generator=g)
    packed = pack_block_fp8(w)
    assert packed.weight.shape == (200, 304) and packed.scale.shape == (2, 3)
    full = packed.weight.float() * _expanded(packed.scale, 128, 200, 304).float()
    assert (full[:, 300:] == 0).all()
    block = w.abs()  # half an E4M3 step (2^-4 of the value, or 2^-10 of the scale below normal)
    step = torch.maximum(block * 2.0 ** -4, _expanded(packed.scale, 128, 200, 300).float() * 2.0 ** -10)
    assert ((full[:, :300] - w).abs() <= step * 1.001).all()
    loaded = block_fp8_weight("w", packed.weight, 1 / packed.scale, inverted=True).to(gpu)
    x = torch.randn(5, 300, generator=g).to(gpu)
    q = quantize_block_rows(x)
    _check(block_fp8_linear(q, loaded, out_dtype=torch.float32), q, loaded)
    with pytest.raises(ValueError):
        block_fp8_weight("w", packed.weight, packed.scale[:1])
    with pytest.raises(ValueError):
        block_fp8_weight("w", packed.weight.float(), packed.scale)


def test_refusals(gpu):
    x, w = _operands(gpu, 4, 256, 96, 1)
    q = quantize_block_rows(x)
    with pytest.raises(N.OmniCodecError):
        quantize_block_rows(x.cpu())
    with pytest.raises(ValueError):
        quantize_block_rows(x.t())
    with pytest.raises(ValueError):
        quantize_block_rows(x.double())
    with pytest.raises(ValueError):
        block_fp8_linear(x[:, :128], w)  # features that the weight does not take
    with pytest.raises(ValueError):
        block_fp8_linear(BlockFp8Rows(q.values, q.scale[:, :1]), w)
    with pytest.raises(ValueError):
        block_fp8_linear(q, BlockFp8Weight(w.weight, w.scale[:, :1]))
    with pytest.raises(ValueError):
        block_fp8_linear(q, w, torch.empty(4, 97, device=gpu))
    with pytest.raises(ValueError):
        block_fp8_linear(q, w, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        block_fp8_linear(q, BlockFp8Weight(w.weight, w.scale, torch.zeros(95, device=gpu)))
    shifted = torch.zeros(4 * 256 + 16, dtype=torch.uint8, device=gpu)[1:1025].view(4, 256)
    with pytest.raises(N.OmniCodecError) as refused:  # rows off the 16-byte grid
        block_fp8_linear(BlockFp8Rows(shifted.view(torch.float8_e4m3fn), q.scale), w)
    assert refused.value.status == N.INVALID_ARG
    with pytest.raises(N.OmniCodecError) as refused:  # features off the 16-byte grid
        block_fp8_linear(BlockFp8Rows(q.values[:, :250], q.scale), BlockFp8Weight(w.weight[:, :250], w.scale))
    assert refused.value.status == N.INVALID_ARG
    with pytest.raises(N.OmniCodecError) as refused:  # one row expanded over four
        block_fp8_linear(BlockFp8Rows(q.values[:1].expand(4, 256), q.scale), w)
    assert refused.value.status == N.INVALID_ARG
