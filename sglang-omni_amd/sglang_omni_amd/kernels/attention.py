"""Attention over a talker's whole context: of prompts, packed sequences of their own lengths, and of one
new token of each stream over its paged key-value cache. Heads are grouped over key heads; scores,
maxima and sums are float32."""

from __future__ import annotations

import torch

from .. import _native as N
from .kv_cache import PagedKvCache

_HALVES = (torch.bfloat16, torch.float16)
_INDEXES = (torch.int64, torch.int32)
_E4M3 = torch.float8_e4m3fn
_CODES = N.TORCH_TO_OMNI
_prompt = _plan = None  # the entry points, bound at the first call
_paged = _workspace = None


def _heads(t: torch.Tensor, name: str) -> tuple[int, int]:
    """The row and head strides of [rows, heads, dim] with 16-byte aligned heads."""
    strides = t.stride()
    if len(strides) != 3 or strides[2] != 1 or strides[0] % 8 or strides[1] % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name} must be [rows, heads, dim] with contiguous, 16-byte aligned heads")
    return strides[0], strides[1]


def _scale(scale: float | None, dim: int) -> float:
    if scale is None:
        return dim ** -0.5
    if not 0.0 < scale <= 1e30:
        raise ValueError(f"scale must be positive, got {scale}")
    return scale


def _starts(t: torch.Tensor, name: str, index: int) -> None:
    if t.get_device() != index or t.dim() != 1 or t.shape[0] < 1 or t.dtype not in _INDEXES \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 or int64 [sequences + 1] on q's GPU")


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, *,
                     key_starts: torch.Tensor | None = None, causal: bool = True,
                     scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of packed sequences, on the current stream: sequence s has the queries
    starts[s] .. starts[s + 1] - 1 of q [tokens, heads, dim] and the keys key_starts[s] .. key_starts[s +
    1] - 1 (starts without it) of k and v [key_tokens, kv_heads, dim]; query head h reads key head h //
    (heads // kv_heads). Starts are int32 / int64 in device memory, ascending; the host does not read
    them.

    Causal: a sequence's last query sees all of its keys, each one before it one key less, so the queries
    may be the last piece of a longer sequence. A query that sees no key (or whose scores are all
    -infinity) is zero, one that sees a NaN score is NaN, and what lies behind a query's keys does not
    reach it, not even as NaN. scale defaults to dim ** -0.5. Softmax weights are rounded to the type before they meet the values, as the
    matrix cores take them; all sums are float32 and the output is rounded once. How a row's keys are
    divided over the chip follows from the call's sizes, and with it the row's last bits.

    bf16 or f16; dim a multiple of 8 up to 256; heads contiguous and 16-byte aligned, other strides free (of
    k and v up to 2^23 between tokens); tokens * (heads // kv_heads) and key_tokens below 2^31 - 255.
    Rows of ``out`` in front of the first sequence and behind the last one stay as they are; those of an
    output made here are zero."""
    index = q.get_device()
    if index < 0 or k.get_device() != index or v.get_device() != index:
        N.require_device(q, k, v)
        raise ValueError("q, k and v must be on one GPU")
    q_token, q_head = _heads(q, "q")
    k_token, k_head = _heads(k, "k")
    v_token, v_head = _heads(v, "v")
    (tokens, heads, dim), (key_tokens, kv_heads, k_dim), dtype = q.shape, k.shape, q.dtype
    if dtype not in _HALVES or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v must be bf16 or f16, of one type")
    if kv_heads < 1 or heads < 1 or heads % kv_heads or k_dim != dim or v.shape != k.shape:
        raise ValueError("k and v must be [key_tokens, kv_heads, dim], kv_heads a divisor of q's heads")
    if dim % 8 or not 8 <= dim <= 256:
        raise ValueError(f"heads must be a multiple of 8 values up to 256, got {dim}")
    _starts(starts, "starts", index)
    if key_starts is None:
        key_starts = starts
    else:
        _starts(key_starts, "key_starts", index)
        if key_starts.shape != starts.shape or key_starts.dtype is not starts.dtype:
            raise ValueError("key_starts must be like starts")
    clear = out is None
    if clear:
        out = torch.empty(tokens, heads, dim, dtype=dtype, device=q.device)
        out_token, out_head = heads * dim, dim
    else:
        out_token, out_head = _heads(out, "out")
        if out.shape != q.shape or out.dtype is not dtype or out.get_device() != index:
            raise ValueError("out must be like q")
    sequences = starts.shape[0] - 1
    global _prompt, _plan
    if _prompt is None:
        lib = N.load_library()
        _prompt, _plan = lib.omni_prompt_attention, lib.omni_prompt_plan
    splits = _plan(tokens, key_tokens, sequences, heads, kv_heads, dim, 1 if causal else 0, None)
    needed = splits * tokens * heads * (dim + 2) * 4 if splits > 1 else 0
    workspace = torch.empty(needed, dtype=torch.uint8, device=q.device) if needed else None
    args = N.pack_prompt(
        q.data_ptr(), q_token, q_head, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head,
        out.data_ptr(), out_token, out_head, _CODES[dtype], tokens, key_tokens, heads, kv_heads, dim,
        starts.data_ptr(), key_starts.data_ptr(), _CODES[starts.dtype], sequences,
        1 if causal else 0, _scale(scale, dim), 1 if clear else 0,
        0 if workspace is None else workspace.data_ptr(), needed)
    status = N.launch_on(index, _prompt, args)
    if status:
        N.check(status, "omni_prompt_attention")
    return out


def paged_attention(q: torch.Tensor, cache: PagedKvCache, table: torch.Tensor, lengths: torch.Tensor,
                    *, scale: float | None = None, max_length: int | None = None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of one query of each sequence, q [batch, heads, dim], over the first
    lengths[b] (int32 / int64 [batch]) keys and values of its cache, on the current stream: key j lies on
    page table[b, j // page_size] (int32 [batch, columns], rows of any stride), place j % page_size. Query
    head h reads key head h // (heads // kv_heads). The lengths stay on the GPU; ``max_length`` is a bound
    on them that the host knows (the table's room without it; longer ones count as it), and the closer it
    is the fewer idle workgroups and the less workspace a call takes.

    A sequence without keys is zero, and so is a row whose scores are all -infinity; a NaN among the scores
    makes the row NaN. Keys on pages outside the cache are left out. The cache holds q's type (bf16 or f16)
    or E4M3, whose rows count their scale times the bytes; scale defaults to dim ** -0.5. A row's bits depend on its own sequence alone, not on the batch beside it nor on max_length."""
    index = q.get_device()
    if index < 0 or cache.index != index or table.get_device() != index \
            or lengths.get_device() != index:
        N.require_device(q, table, lengths)
        raise ValueError("q, the cache, table and lengths must be on one GPU")
    q_row, q_head = _heads(q, "q")
    (batch, heads, dim), dtype = q.shape, q.dtype
    if dtype not in _HALVES or (cache.dtype is not dtype and cache.dtype is not _E4M3):
        raise ValueError("q must be bf16 or f16, and the cache of its type or E4M3")
    if dim != cache.dim or heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"q must be [batch, heads, {cache.dim}], heads a multiple of {cache.kv_heads}")
    if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != batch \
            or (table.stride(1) != 1 and table.shape[1] > 1):
        raise ValueError(f"table must be int32 [{batch}, columns] with contiguous rows")
    if lengths.dtype not in _INDEXES or lengths.dim() != 1 or lengths.shape[0] != batch \
            or not lengths.is_contiguous():
        raise ValueError(f"lengths must be contiguous int32 or int64 [{batch}]")
    columns = table.shape[1]
    room = columns * cache.page_size
    if max_length is None:
        max_length = room
    elif max_length < 0:
        raise ValueError(f"max_length must not be negative, got {max_length}")
    max_length = min(max_length, room)
    if out is None:
        out = torch.empty(batch, heads, dim, dtype=dtype, device=q.device)
        out_row, out_head = heads * dim, dim
    else:
        out_row, out_head = _heads(out, "out")
        if out.shape != q.shape or out.dtype is not dtype or out.get_device() != index:
            raise ValueError("out must be like q")
    global _paged, _workspace
    if _paged is None:
        lib = N.load_library()
        _paged, _workspace = lib.omni_paged_attention, lib.omni_paged_workspace
    needed = _workspace(batch, heads, cache.kv_heads, dim, max_length)
    workspace = torch.empty(needed, dtype=torch.uint8, device=q.device) if needed else None
    args = N.pack_paged(
        q.data_ptr(), q_row, q_head, out.data_ptr(), out_row, out_head, _CODES[dtype], batch, heads,
        cache.address, table.data_ptr(), table.stride(0), columns, lengths.data_ptr(),
        _CODES[lengths.dtype], max_length, _scale(scale, dim),
        0 if workspace is None else workspace.data_ptr(), needed)
    status = N.launch_on(index, _paged, args)
    if status:
        N.check(status, "omni_paged_attention")
    return out


__all__ = ["paged_attention", "prompt_attention"]
