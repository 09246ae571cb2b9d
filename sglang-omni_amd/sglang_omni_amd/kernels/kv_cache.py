"""The paged key-value cache of a talker's streams: rows of keys and values on pages of a fixed number
of tokens, in bf16 or f16 as they are or in 8-bit floating point (OCP E4M3) with a float32 scale per row
and head. A token's slot is page * page_size + its place on the page; a stream's pages are in any order,
listed in its row of a page table."""

from __future__ import annotations

import ctypes

import torch

from .. import _native as N

_E4M3 = torch.float8_e4m3fn
_FLOATS = (torch.bfloat16, torch.float16, torch.float32)
_HELD = (torch.bfloat16, torch.float16, _E4M3)
_INDEXES = (torch.int64, torch.int32)
_CODES = N.TORCH_TO_OMNI
_read = None  # the entry points, bound at the first call
_write = None


class PagedKvCache:
    """keys and values [pages, kv_heads, page_size, dim] of bf16, f16 or E4M3 (``torch.float8_e4m3fn``)
    and the same strides, dim contiguous and a multiple of 16 up to 256, rows 16-byte aligned (pages with
    their tokens outside the heads are taken as transposed views); with E4M3 their float32 scales
    [pages, kv_heads, page_size]. The tensors are held as they are, and not replaced afterwards."""

    __slots__ = ("_keys", "_values", "_key_scale", "_value_scale", "_struct", "address", "index",
                 "pages", "kv_heads", "page_size", "dim", "dtype")

    def __init__(self, keys: torch.Tensor, values: torch.Tensor,
                 key_scale: torch.Tensor | None = None, value_scale: torch.Tensor | None = None):
        index = keys.get_device()
        if index < 0 or values.get_device() != index:
            N.require_device(keys, values)
            raise ValueError("keys and values must be on one GPU")
        dtype, shape, strides = keys.dtype, keys.shape, keys.stride()
        if dtype not in _HELD or len(shape) != 4:
            raise ValueError("keys must be bf16, f16 or E4M3 [pages, kv_heads, page_size, dim]")
        if values.dtype is not dtype or values.shape != shape or values.stride() != strides:
            raise ValueError("values must be like keys, strides too")
        pages, kv_heads, page_size, dim = shape
        if pages < 1 or kv_heads < 1 or page_size < 1 or dim % 16 or not 16 <= dim <= 256:
            raise ValueError("a cache has pages, heads and tokens, and heads of a multiple of 16 up to 256")
        if pages * page_size > 0x7fffffff:
            raise ValueError("a cache has at most 2^31 - 1 slots")
        each = 16 if dtype is _E4M3 else 8
        if strides[3] != 1 or strides[0] % each or strides[1] % each or strides[2] % each \
                or keys.data_ptr() % 16 or values.data_ptr() % 16:
            raise ValueError("a cache's rows must be contiguous and 16-byte aligned")
        if dtype is _E4M3:
            if key_scale is None or value_scale is None or key_scale.dtype is not torch.float32 \
                    or value_scale.dtype is not torch.float32 or key_scale.get_device() != index \
                    or value_scale.get_device() != index or key_scale.shape != shape[:3] \
                    or value_scale.shape != shape[:3] or key_scale.stride() != value_scale.stride():
                raise ValueError(f"an E4M3 cache has float32 scales {list(shape[:3])} of the same "
                                 "strides for keys and values")
            scales = (key_scale.data_ptr(), value_scale.data_ptr(), *key_scale.stride())
        elif key_scale is None and value_scale is None:
            scales = (0, 0, 0, 0, 0)
        else:
            raise ValueError("scales go with E4M3 rows")
        self._keys, self._values = keys, values
        self._key_scale, self._value_scale = key_scale, value_scale
        self.index, self.dtype = index, dtype
        self.pages, self.kv_heads, self.page_size, self.dim = pages, kv_heads, page_size, dim
        packed = N.pack_kv_cache(keys.data_ptr(), values.data_ptr(), _CODES[dtype], *strides[:3],
                                 *scales, pages, page_size, kv_heads, dim)
        self._struct = ctypes.create_string_buffer(packed, len(packed))
        self.address = ctypes.addressof(self._struct)

    keys = property(lambda self: self._keys)
    values = property(lambda self: self._values)
    key_scale = property(lambda self: self._key_scale)
    value_scale = property(lambda self: self._value_scale)

    @classmethod
    def allocate(cls, pages: int, page_size: int, kv_heads: int, dim: int,
                 dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda") -> "PagedKvCache":
        """A cache of zeros; a head's tokens lie side by side on a page."""
        if dtype not in _HELD:
            raise ValueError("a cache holds bf16, f16 or E4M3")
        shape = (pages, kv_heads, page_size, dim)
        rows = [torch.zeros(shape, dtype=torch.uint8 if dtype is _E4M3 else dtype, device=device)
                for _ in range(2)]
        if dtype is not _E4M3:
            return cls(*rows)
        return cls(*(t.view(_E4M3) for t in rows),
                   *(torch.ones(shape[:3], device=device) for _ in range(2)))


def _rows(t: torch.Tensor, name: str, cache: PagedKvCache) -> tuple[int, int]:
    """The token and head strides of [tokens, kv_heads, dim] rows."""
    shape, strides = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != cache.kv_heads or shape[2] != cache.dim or strides[2] != 1:
        raise ValueError(f"{name} must be [tokens, {cache.kv_heads}, {cache.dim}] with contiguous dim")
    return strides[0], strides[1]


def _slots(slots: torch.Tensor, tokens: int, index: int) -> tuple[int, int, int]:
    """The address, type and stride of the slots of `tokens` tokens."""
    if slots.get_device() != index or slots.dim() != 1 or slots.shape[0] != tokens \
            or slots.dtype not in _INDEXES:
        raise ValueError(f"slots must be int32 or int64 [{tokens}] on the cache's GPU")
    return slots.data_ptr(), _CODES[slots.dtype], slots.stride(0)


def write_kv_cache(cache: PagedKvCache, k: torch.Tensor, v: torch.Tensor,
                   slots: torch.Tensor) -> None:
    """k and v [tokens, kv_heads, dim] (bf16, f16 or f32, any strides with contiguous dim) into the
    cache's rows of slots [tokens] (int32 / int64), on the current stream. 16-bit caches take the values
    rounded to their type; an E4M3 cache each head's row with scale = max|row| / 448 (1 for a row of
    zeros, infinite for a row with an infinity; NaN stays NaN). A token whose slot is not in the cache, a
    padded row's -1 for instance, is passed over. Slots must differ: of two tokens with one slot the row
    holds any mix."""
    index = cache.index
    if k.get_device() != index or v.get_device() != index:
        N.require_device(k, v)
        raise ValueError("k, v and the cache must be on one GPU")
    k_token, k_head = _rows(k, "k", cache)
    v_token, v_head = _rows(v, "v", cache)
    tokens, dtype = k.shape[0], k.dtype
    if dtype not in _FLOATS or v.dtype is not dtype or v.shape[0] != tokens:
        raise ValueError("k and v must be bf16, f16 or f32, of one type and number of tokens")
    args = N.pack_norm_rotary(
        0, 0, 0, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, 0, 0, 0, 0, 0, 0,
        _CODES[dtype], tokens, 0, cache.kv_heads, cache.dim, 0, 0, 0, 0.0, 0, 0, 0, 0, 0, 1.0,
        N.ROTARY_HALF, cache.address, *_slots(slots, tokens, index))
    global _write
    if _write is None:
        _write = N.load_library().omni_norm_rotary
    status = N.launch_on(index, _write, args)
    if status:
        N.check(status, "omni_norm_rotary")


def _read_into(t: torch.Tensor, name: str, tokens: int, dtype: torch.dtype,
               cache: PagedKvCache) -> tuple[int, int]:
    strides = _rows(t, name, cache)
    if t.shape[0] != tokens or t.dtype is not dtype or t.get_device() != cache.index:
        raise ValueError(f"{name} must be [{tokens}, {cache.kv_heads}, {cache.dim}] of {dtype} on the "
                         "cache's GPU")
    return strides


def read_kv_cache(cache: PagedKvCache, slots: torch.Tensor, *, dtype: torch.dtype | None = None,
                  k_out: torch.Tensor | None = None, v_out: torch.Tensor | None = None
                  ) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values [tokens, kv_heads, dim] of slots [tokens] (int32 / int64), on the current
    stream, as dtype (bf16, f16 or f32; the cache's own, bf16 for E4M3), rounded once. A slot that is not
    in the cache gives zeros. What a prompt's next piece attends to, for instance."""
    index = cache.index
    if slots.get_device() != index:
        N.require_device(slots)
        raise ValueError("slots and the cache must be on one GPU")
    if dtype is None:
        given = k_out if k_out is not None else v_out
        dtype = given.dtype if given is not None else \
            torch.bfloat16 if cache.dtype is _E4M3 else cache.dtype
    if dtype not in _FLOATS:
        raise ValueError("rows are read as bf16, f16 or f32")
    tokens = slots.shape[0] if slots.dim() == 1 else -1
    slots_ptr, slots_dtype, slots_stride = _slots(slots, tokens, index)
    kv_heads, dim = cache.kv_heads, cache.dim
    k_token = v_token = kv_heads * dim
    k_head = v_head = dim
    if k_out is None:
        k_out = torch.empty(tokens, kv_heads, dim, dtype=dtype, device=slots.device)
    else:
        k_token, k_head = _read_into(k_out, "k_out", tokens, dtype, cache)
    if v_out is None:
        v_out = torch.empty(tokens, kv_heads, dim, dtype=dtype, device=slots.device)
    else:
        v_token, v_head = _read_into(v_out, "v_out", tokens, dtype, cache)
    args = N.pack_read_cache(cache.address, slots_ptr, slots_dtype, slots_stride, tokens,
                             k_out.data_ptr(), k_token, k_head, v_out.data_ptr(), v_token, v_head,
                             _CODES[dtype])
    global _read
    if _read is None:
        _read = N.load_library().omni_read_cache
    status = N.launch_on(index, _read, args)
    if status:
        N.check(status, "omni_read_cache")
    return k_out, v_out


__all__ = ["PagedKvCache", "read_kv_cache", "write_kv_cache"]
