"""Logit adjustments against a row-by-row float64 loop: every part alone and together, vocabularies
around the tile, histories of every length, repeated and foreign ids, masks that leave nothing,
slots, strides and non-finite logits."""

from __future__ import annotations

import math

import pytest
import torch

from sglang_omni_amd import _native as N
from sglang_omni_amd.kernels import adjust_logits

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}


def _reference(logits, kw):
    """The definition in Python, and per element the magnitude its float32 steps round at."""
    rows, vocab = logits.shape
    out = logits.double().cpu()
    size = torch.where(out.isfinite(), out.abs(), torch.zeros_like(out))
    kw = {k: (v.cpu() if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
    for r in range(rows):
        if kw.get("history") is not None:
            slot = int(kw["slot_index"][r]) if kw.get("slot_index") is not None else r
            tokens, prompt = [], 0
            if 0 <= slot < kw["history"].shape[0]:
                length = max(0, min(int(kw["lengths"][slot]), kw["history"].shape[1]))
                tokens = kw["history"][slot, :length].tolist()
                prompt = int(kw["prompt_lengths"][slot]) if kw.get("prompt_lengths") is not None else 0
            seen, count = set(), {}
            for i, t in enumerate(tokens):
                if 0 <= t < vocab:
                    seen.add(t)
                    if i >= prompt:
                        count[t] = count.get(t, 0) + 1
            if kw.get("repetition") is not None:
                rep = float(kw["repetition"][r])
                for t in seen:
                    v = float(out[r, t])
                    out[r, t] = v / rep if v > 0 else v * rep
                    size[r, t] *= max(rep, 1 / rep)
            for t, n in count.items():
                f = float(kw["frequency"][r]) if kw.get("frequency") is not None else 0.0
                p = float(kw["presence"][r]) if kw.get("presence") is not None else 0.0
                out[r, t] -= f * n + p
                size[r, t] += abs(f) * n + abs(p)
        if kw.get("bias_tokens") is not None:
            last = {}
            for t, v in zip(kw["bias_tokens"][r].tolist(), kw["bias_values"][r].tolist()):
                if 0 <= t < vocab:
                    last[t] = v
            for t, v in last.items():
                out[r, t] += v
                size[r, t] += abs(v)
        if kw.get("allowed") is not None:
            m = int(kw["allowed_index"][r]) if kw.get("allowed_index") is not None else r
            if 0 <= m < kw["allowed"].shape[0]:
                words = kw["allowed"][m].tolist()
                bits = torch.tensor([(words[v >> 5] >> (v & 31)) & 1 for v in range(vocab)])
                out[r, bits == 0] = -math.inf
    return out, size


def _check(logits, **kw):
    """At most six float32 roundings of the magnitudes that meet in an element, then one rounding to
    the output's type."""
    got = adjust_logits(logits, **{k: v for k, v in kw.items()})
    want, size = _reference(logits, kw)
    got64 = got.double().cpu()
    assert torch.equal(got64.isfinite(), want.isfinite())
    assert torch.equal(got64.isnan(), want.isnan())
    odd = ~want.isfinite() & ~want.isnan()
    assert torch.equal(got64[odd], want[odd])
    fine = want.isfinite()
    bound = 6 * 2.0 ** -24 * size + HALF_ULP[got.dtype] * want.abs() + 2.0 ** -25
    assert ((got64 - want).abs()[fine] <= bound[fine]).all()
    return got


def _inputs(gpu, rows, vocab, capacity, seed, ints=torch.int32):
    g = torch.Generator().manual_seed(seed)
    kw = {
        "history": (torch.rand(rows, capacity, generator=g) ** 2 * vocab).to(ints),
        "lengths": torch.randint(0, capacity + 1, (rows,), generator=g),
        "prompt_lengths": torch.randint(0, capacity + 1, (rows,), generator=g),
        "repetition": 0.7 + torch.rand(rows, generator=g),
        "frequency": torch.rand(rows, generator=g) - 0.3,
        "presence": torch.rand(rows, generator=g) - 0.3,
        "bias_tokens": torch.randint(-1, vocab, (rows, 7), generator=g).to(ints),
        "bias_values": torch.randn(rows, 7, generator=g) * 5,
        "allowed": torch.randint(-2**31, 2**31, (rows, -(-vocab // 32)), generator=g).to(torch.int32),
    }
    logits = torch.randn(rows, vocab, generator=g) * 4
    return logits.to(gpu), {k: v.to(gpu) for k, v in kw.items()}


PENALTIES = ("repetition", "frequency", "presence")
HISTORY = ("history", "lengths", "prompt_lengths")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("vocab", [1, 31, 33, 1000, 2048, 4095, 4096, 4097, 9001])
def test_everything_together(gpu, dtype, vocab):
    for rows, capacity, ints in ((1, 1, torch.int32), (3, 300, torch.int64), (5, 1000, torch.int32)):
        logits, kw = _inputs(gpu, rows, vocab, capacity, vocab + rows, ints)
        _check(logits.to(dtype), **kw)


@pytest.mark.parametrize("parts", [
    (), HISTORY[:2], (*HISTORY, "repetition"), (*HISTORY, "frequency"), (*HISTORY[:2], "presence"),
    ("bias_tokens", "bias_values"), ("allowed",), ("allowed", "bias_tokens", "bias_values"),
    (*HISTORY, *PENALTIES)])
def test_each_part_alone(gpu, parts):
    logits, kw = _inputs(gpu, 4, 5000, 200, 11)
    got = _check(logits, **{k: kw[k] for k in parts})
    if not set(parts) & {*PENALTIES, "allowed", "bias_tokens"}:
        assert torch.equal(got, logits)


def test_slots_and_foreign_ids(gpu):
    logits, kw = _inputs(gpu, 6, 700, 90, 3)
    kw["history"][0, :5] = torch.tensor([-1, 700, 2**31 - 1, -2**31, 699], device=gpu)
    kw["lengths"][0], kw["prompt_lengths"][0] = 90, 0
    kw["lengths"][1] = 10**9  # past the capacity: clamped
    kw["lengths"][2] = -5     # nothing
    kw["prompt_lengths"][3] = 10**9
    kw["slot_index"] = torch.tensor([0, 1, 2, 3, 6, -1], device=gpu)
    kw["allowed_index"] = torch.tensor([5, 5, -1, 6, 0, 1], device=gpu)
    kw["bias_tokens"][0] = 5
    kw["bias_tokens"][1, :3] = torch.tensor([2**31 - 1, -7, 700], device=gpu)
    _check(logits, **kw)
    wide = {k: v.long() if k in ("history", "bias_tokens") else v for k, v in kw.items()}
    wide["history"][0, 0] = 2**40
    wide["bias_tokens"][1, 0] = -2**40
    _check(logits, **wide)


def test_masks_that_leave_little_or_nothing(gpu):
    logits, kw = _inputs(gpu, 3, 4500, 50, 7)
    kw["allowed"][0] = 0
    kw["allowed"][1] = 0
    kw["allowed"][1, 4499 // 32] = 1 << (4499 % 32)
    got = _check(logits, **kw)
    assert (got[0] == -math.inf).all()
    assert got[1].isfinite().nonzero().flatten().tolist() == [4499]


def test_non_finite_logits(gpu):
    """Infinities follow the formula, NaN stays, and what the mask forbids is -infinity all the same."""
    logits, kw = _inputs(gpu, 2, 300, 40, 9)
    kw["frequency"], kw["presence"] = kw["frequency"].abs(), kw["presence"].abs()
    logits[:, 0:40:4], logits[:, 1:40:4] = math.inf, -math.inf
    logits[:, 2:40:4] = math.nan
    logits[:, 3:40:4] = torch.finfo(F32).min
    kw["history"] = torch.arange(40, device=gpu, dtype=torch.int32).expand(2, 40).contiguous()
    kw["lengths"] = torch.tensor([40, 40], device=gpu)
    kw["prompt_lengths"] = torch.tensor([0, 20], device=gpu)
    kw["repetition"] = torch.tensor([1.0, 0.5], device=gpu)
    kw["bias_tokens"] = torch.full_like(kw["bias_tokens"], -1)
    _check(logits, **kw)


def test_long_history_counts(gpu):
    """One token made 70 000 times, another once."""
    logits = torch.zeros(1, 64, device=gpu)
    history = torch.full((1, 70001), 9, dtype=torch.int32, device=gpu)
    history[0, 70000] = 3
    got = adjust_logits(logits, history=history, lengths=torch.tensor([70001], device=gpu),
                        frequency=torch.tensor([0.5], device=gpu),
                        presence=torch.tensor([0.25], device=gpu))
    want = torch.zeros(1, 64, device=gpu)
    want[0, 9], want[0, 3] = -35000.25, -0.75
    assert torch.equal(got, want)


@pytest.mark.parametrize("entries", [1, 63, 65, 130, 600, 1100])
@pytest.mark.parametrize("vocab", [40, 9001, 20000])
def test_long_bias_lists_with_repeats(gpu, entries, vocab):
    """Lists shorter and longer than a wave and than a workgroup; most tokens named several times."""
    g = torch.Generator().manual_seed(entries + vocab)
    logits, kw = _inputs(gpu, 2, vocab, 300, entries)
    tokens = torch.randint(-1, min(vocab, 200), (2, entries), generator=g)
    tokens[1] *= max(1, vocab // 200)
    kw["bias_tokens"] = tokens.to(torch.int32).to(gpu)
    kw["bias_values"] = (torch.randn(2, entries, generator=g) * 5).to(gpu)
    _check(logits, **kw)


def test_strides_outputs_and_in_place(gpu):
    logits, kw = _inputs(gpu, 5, 3001, 64, 13)
    want = adjust_logits(logits, **kw)
    wide = torch.zeros(5, 3100, device=gpu)[:, 1:3002].copy_(logits)
    strided = {**kw, "history": torch.zeros(5, 100, dtype=torch.int32, device=gpu)[:, 3:67].copy_(kw["history"]),
               "allowed": torch.zeros(5, 99, dtype=torch.int32, device=gpu)[:, :94].copy_(kw["allowed"])}
    buffer = torch.full((6, 3050), math.nan, device=gpu)
    got = adjust_logits(wide, out=buffer[:5, 7:3008], **strided)
    assert torch.equal(got, want)
    assert buffer[5].isnan().all() and buffer[:, :7].isnan().all() and buffer[:, 3008:].isnan().all()
    half = adjust_logits(logits.to(BF16), out=torch.empty(5, 3001, device=gpu), **kw)
    assert torch.equal(half.to(BF16), adjust_logits(logits.to(BF16), **kw))
    assert adjust_logits(logits, out=logits, **kw).data_ptr() == logits.data_ptr()
    assert torch.equal(logits, want)
    assert adjust_logits(logits[:0]).shape == (0, 3001)


def test_refusals(gpu):
    logits, kw = _inputs(gpu, 3, 500, 20, 1)
    history = {k: kw[k] for k in HISTORY}
    bad = [
        {"lengths": kw["lengths"]}, {"history": kw["history"]}, {"repetition": kw["repetition"]},
        {**history, "repetition": kw["repetition"][:2]}, {**history, "repetition": kw["repetition"].double()},
        {**history, "lengths": kw["lengths"][:2]}, {**history, "lengths": kw["lengths"].float()},
        {**history, "prompt_lengths": kw["prompt_lengths"].int()},
        {**history, "history": kw["history"].float()},
        {"history": kw["history"][:2], "lengths": kw["lengths"][:2]},
        {**history, "slot_index": torch.zeros(3, dtype=torch.int32, device=gpu)},
        {"bias_tokens": kw["bias_tokens"]},
        {"bias_tokens": kw["bias_tokens"], "bias_values": kw["bias_values"][:, :3]},
        {**history, "bias_tokens": kw["bias_tokens"].long(), "bias_values": kw["bias_values"]},
        {"allowed": kw["allowed"][:, :15]}, {"allowed": kw["allowed"].long()},
        {"allowed": kw["allowed"][:2]}, {"allowed_index": torch.zeros(3, dtype=torch.int64, device=gpu)},
        {"out": torch.empty(3, 499, device=gpu)}, {"out": torch.empty(3, 500, device=gpu, dtype=BF16)},
    ]
    for case in bad:
        with pytest.raises(ValueError):
            adjust_logits(logits, **case)
    with pytest.raises(ValueError):
        adjust_logits(logits.double())
    with pytest.raises(ValueError):
        adjust_logits(logits.t())
    with pytest.raises(N.OmniCodecError):
        adjust_logits(logits.cpu())
