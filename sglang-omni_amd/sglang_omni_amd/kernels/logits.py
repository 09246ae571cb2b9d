"""What a sampler does to logits before it draws from them, in one launch: penalties for the tokens
of a row's history, its bias list, and its grammar's mask."""

from __future__ import annotations

import torch

from .. import _native as N

_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_CODES, _pack, _raw_stream = N.TORCH_TO_OMNI, N.pack_logits, N.raw_stream
_launch = None  # the entry point, bound at the first call
_INTS = (torch.int32, torch.int64)


def _per_row(t: torch.Tensor | None, rows: int, dtype: torch.dtype, what: str, index: int) -> int:
    """The address of a per-row vector on GPU ``index``, 0 for none."""
    if t is None:
        return 0
    if t.get_device() != index or t.dtype is not dtype or t.numel() != rows \
            or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {dtype} [{rows}] on the logits' GPU")
    return t.data_ptr()


def _row_stride(t: torch.Tensor, what: str, index: int) -> int:
    """The row stride of a matrix with contiguous rows on GPU ``index``."""
    strides = t.stride()
    if t.get_device() != index or len(strides) != 2:
        raise ValueError(f"{what} must be a matrix on the logits' GPU")
    rows, width = t.shape
    if strides[1] != 1 and width > 1:
        raise ValueError(f"{what} must have contiguous rows")
    return strides[0] if rows > 1 else width


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
    index = logits.get_device()
    if index < 0:
        N.require_device(logits)
    dtype = logits.dtype
    if dtype not in _FLOATS:
        raise ValueError("logits must be f32, bf16 or f16")
    stride = _row_stride(logits, "logits", index)
    rows, vocab = logits.shape
    if vocab < 1:
        raise ValueError("logits have no vocabulary")
    if out is None:
        out = torch.empty_like(logits)
        out_dtype, out_stride = dtype, N.row_stride(out)
    else:
        out_dtype = out.dtype
        if out.shape != logits.shape or (out_dtype is not dtype and out_dtype is not torch.float32):
            raise ValueError("out must be like the logits, or float32")
        out_stride = _row_stride(out, "out", index)
    tokens_dtype = lengths_dtype = torch.int32
    history_ptr = history_stride = capacity = slots = lengths_ptr = prompt_ptr = 0
    if history is None:
        if not (lengths is None and prompt_lengths is None and slot_index is None
                and repetition is None and frequency is None and presence is None):
            raise ValueError("lengths, slots and penalties go with a history")
    else:
        history_stride = _row_stride(history, "history", index)
        slots, capacity = history.shape
        tokens_dtype = history.dtype
        if tokens_dtype not in _INTS or lengths is None or lengths.dtype not in _INTS:
            raise ValueError("history must be int32 or int64 and come with lengths of such a dtype")
        lengths_dtype = lengths.dtype
        lengths_ptr = _per_row(lengths, slots, lengths_dtype, "lengths", index)
        prompt_ptr = _per_row(prompt_lengths, slots, lengths_dtype, "prompt_lengths", index)
        if slot_index is None and slots < rows:
            raise ValueError(f"{slots} histories for {rows} rows need a slot_index")
        history_ptr = history.data_ptr()
    bias_ptr = values_ptr = biases = tokens_stride = values_stride = 0
    if bias_tokens is not None and bias_values is not None:
        tokens_stride = _row_stride(bias_tokens, "bias_tokens", index)
        values_stride = _row_stride(bias_values, "bias_values", index)
        bias_dtype = bias_tokens.dtype
        if (bias_tokens.shape != bias_values.shape or bias_tokens.shape[0] != rows
                or bias_values.dtype is not torch.float32 or bias_dtype not in _INTS
                or (history is not None and bias_dtype is not tokens_dtype)):
            raise ValueError("bias_tokens (int32 or int64, as the history) and bias_values "
                             "(float32) must be [rows, entries] alike")
        tokens_dtype = bias_dtype
        biases = bias_tokens.shape[1]
        bias_ptr, values_ptr = bias_tokens.data_ptr(), bias_values.data_ptr()
    elif bias_tokens is not None or bias_values is not None:
        raise ValueError("bias_tokens and bias_values come together")
    allowed_ptr = masks = allowed_stride = 0
    if allowed is not None:
        allowed_stride = _row_stride(allowed, "allowed", index)
        masks, words = allowed.shape
        if allowed.dtype is not torch.int32 or words < (vocab + 31) // 32:
            raise ValueError(f"allowed must be int32 [masks, {(vocab + 31) // 32}]")
        if allowed_index is None and masks < rows:
            raise ValueError(f"{masks} masks for {rows} rows need an allowed_index")
        allowed_ptr = allowed.data_ptr()
    elif allowed_index is not None:
        raise ValueError("allowed_index goes with allowed")
    f32, i64 = torch.float32, torch.int64
    args = _pack(
        logits.data_ptr(), _CODES[dtype], stride, out.data_ptr(), _CODES[out_dtype], out_stride, rows,
        vocab, history_ptr, _CODES[tokens_dtype], history_stride, capacity, slots, lengths_ptr,
        prompt_ptr, _CODES[lengths_dtype], _per_row(slot_index, rows, i64, "slot_index", index),
        _per_row(repetition, rows, f32, "repetition", index),
        _per_row(frequency, rows, f32, "frequency", index),
        _per_row(presence, rows, f32, "presence", index), bias_ptr, tokens_stride, values_ptr,
        values_stride, biases, allowed_ptr, allowed_stride, masks,
        _per_row(allowed_index, rows, i64, "allowed_index", index))
    global _launch
    if _launch is None:
        _launch = N.load_library().omni_adjust_logits
    status = _launch(args, _raw_stream(index))
    if status:
        N.check(status, "omni_adjust_logits")
    return out


__all__ = ["adjust_logits"]
