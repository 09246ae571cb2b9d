"""What a sampler does to logits before it draws from them, in one launch: penalties for the tokens
of a row's history, its bias list, and its grammar's mask."""

from __future__ import annotations

import ctypes

import torch

from .. import _native as N

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_INTS = (torch.int32, torch.int64)


def _per_row(t: torch.Tensor | None, rows: int, what: str, device: torch.device) -> int | None:
    if t is None:
        return None
    if t.device != device or t.dtype != torch.float32 or t.shape != (rows,) \
            or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous float32 [{rows}] on the logits' GPU")
    return t.data_ptr()


def _row_matrix(t: torch.Tensor, what: str, device: torch.device) -> int:
    """t's row stride, checked to be a matrix of contiguous rows on the logits' GPU."""
    if t.dim() != 2 or t.device != device or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{what} must be a matrix with contiguous rows on the logits' GPU")
    return N.row_stride(t)


def _index(t: torch.Tensor | None, rows: int, what: str, device: torch.device) -> int | None:
    if t is None:
        return None
    if t.device != device or t.dtype != torch.int64 or t.shape != (rows,) or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous int64 [{rows}] on the logits' GPU")
    return t.data_ptr()


def adjust_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None,
                  lengths: torch.Tensor | None = None,
                  prompt_lengths: torch.Tensor | None = None,
                  slot_index: torch.Tensor | None = None,
                  repetition: torch.Tensor | None = None, frequency: torch.Tensor | None = None,
                  presence: torch.Tensor | None = None, bias_tokens: torch.Tensor | None = None,
                  bias_values: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                  allowed_index: torch.Tensor | None = None, out: torch.Tensor | None = None
                  ) -> torch.Tensor:
    """logits [rows, vocab] (f32, bf16, f16) adjusted on the current stream, in this order, in
    float32, rounded once:

    - a token of the row's history: l / repetition where l > 0, else l * repetition
    - one made past the prompt, count times: l - frequency * count - presence
    - the row's bias list: l + bias_values[row, i] for token bias_tokens[row, i] (int32 / int64; a
      negative id is an unused entry; of several entries for one token the last stands)
    - allowed: -infinity where the token's bit is 0 (int32 [masks, ceil(vocab / 32)], token v at bit
      v % 32 of word v // 32); allowed_index [rows] names each row's mask, -1 none, by default its own

    history [slots, capacity] (int32 / int64) holds tokens, lengths [slots] how many of each slot's
    count, prompt_lengths [slots] how many of those are the prompt (none by default); slot_index
    [rows] names each row's slot, by default its own. repetition, frequency and presence are float32
    [rows]. Each part is optional. ``out`` (f32 or the logits' dtype) may be the logits."""
    N.require_device(logits, history, lengths, prompt_lengths, slot_index, repetition, frequency,
                     presence, bias_tokens, bias_values, allowed, allowed_index, out)
    device = logits.device
    if logits.dtype not in _FLOATS:
        raise ValueError("logits must be f32, bf16 or f16")
    stride = _row_matrix(logits, "logits", device)
    rows, vocab = logits.shape
    if vocab < 1:
        raise ValueError("logits have no vocabulary")
    if out is None:
        out = torch.empty(rows, vocab, dtype=logits.dtype, device=device)
    elif out.shape != logits.shape or out.dtype not in (logits.dtype, torch.float32):
        raise ValueError("out must be like the logits, or float32")
    out_stride = _row_matrix(out, "out", device)
    penalties = [_per_row(t, rows, what, device)
                 for t, what in ((repetition, "repetition"), (frequency, "frequency"),
                                 (presence, "presence"))]
    tokens_dtype = lengths_dtype = torch.int32
    history_stride = capacity = slots = 0
    if history is None:
        if any(t is not None for t in (lengths, prompt_lengths, slot_index, *penalties)):
            raise ValueError("lengths, slots and penalties go with a history")
    else:
        history_stride = _row_matrix(history, "history", device)
        slots, capacity = history.shape
        tokens_dtype = history.dtype
        if tokens_dtype not in _INTS or lengths is None:
            raise ValueError("history must be int32 or int64 and come with lengths")
        lengths_dtype = lengths.dtype
        for t, what in ((lengths, "lengths"), (prompt_lengths, "prompt_lengths")):
            if t is not None and (t.dtype not in _INTS or t.dtype != lengths_dtype
                                  or t.shape != (slots,) or not t.is_contiguous()
                                  or t.device != device):
                raise ValueError(f"{what} must be contiguous int32 or int64 [{slots}], both alike")
        if slot_index is None and slots < rows:
            raise ValueError(f"{slots} histories for {rows} rows need a slot_index")
    biases = tokens_stride = values_stride = 0
    if (bias_tokens is None) != (bias_values is None):
        raise ValueError("bias_tokens and bias_values come together")
    if bias_tokens is not None:
        tokens_stride = _row_matrix(bias_tokens, "bias_tokens", device)
        values_stride = _row_matrix(bias_values, "bias_values", device)
        if (bias_tokens.shape != bias_values.shape or bias_tokens.shape[0] != rows
                or bias_values.dtype != torch.float32 or bias_tokens.dtype not in _INTS
                or (history is not None and bias_tokens.dtype != tokens_dtype)):
            raise ValueError("bias_tokens (int32 or int64, as the history) and bias_values "
                             "(float32) must be [rows, entries] alike")
        tokens_dtype = bias_tokens.dtype
        biases = bias_tokens.shape[1]
    masks = allowed_stride = 0
    if allowed is not None:
        allowed_stride = _row_matrix(allowed, "allowed", device)
        masks = allowed.shape[0]
        if allowed.dtype != torch.int32 or allowed.shape[1] < (vocab + 31) // 32:
            raise ValueError(f"allowed must be int32 [masks, {(vocab + 31) // 32}]")
        if allowed_index is None and masks < rows:
            raise ValueError(f"{masks} masks for {rows} rows need an allowed_index")
    elif allowed_index is not None:
        raise ValueError("allowed_index goes with allowed")
    args = N.LogitsArgs(
        logits.data_ptr(), N.omni_dtype(logits.dtype), stride, out.data_ptr(),
        N.omni_dtype(out.dtype), out_stride, rows, vocab, N.ptr(history),
        N.omni_dtype(tokens_dtype), history_stride, capacity, slots, N.ptr(lengths),
        N.ptr(prompt_lengths), N.omni_dtype(lengths_dtype),
        _index(slot_index, rows, "slot_index", device), *penalties, N.ptr(bias_tokens),
        tokens_stride, N.ptr(bias_values), values_stride, biases, N.ptr(allowed), allowed_stride,
        masks, _index(allowed_index, rows, "allowed_index", device))
    lib = N.load_library()
    N.check(lib.omni_adjust_logits(ctypes.byref(args), N.stream_handle(device)),
            "omni_adjust_logits")
    return out


__all__ = ["adjust_logits"]
