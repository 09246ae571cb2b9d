"""Calls of the attention and cache operators whose launch would have 2^32 threads or more are refused
before any launch, without a GPU; the largest ones below are not."""

from __future__ import annotations

from sglang_omni_amd import _native as N
from tests.test_attention_abi import _fields


def _cache(dim=16, **kw):
    struct = N.KvCacheStruct(*_fields(N.KvCacheStruct, keys=4096, values=4096, dtype=N.DTYPE_BF16,
                                      stride_page=256, stride_head=128, stride_token=dim, pages=4, page_size=8,
                                      kv_heads=2, dim=dim, **kw))
    _cache.kept = struct
    return N.ctypes.addressof(struct)


def test_too_many_sequences():
    lib = N.load_library()

    def status(**kw):
        fields = dict(q=4096, k=4096, v=4096, out=4096, dtype=N.DTYPE_BF16, tokens=8, key_tokens=8, heads=1,
                      kv_heads=1, dim=16, starts=4096, key_starts=4096, starts_dtype=N.DTYPE_I32, causal=1,
                      clear_rest=1)
        return lib.omni_prompt_attention(N.pack_prompt(*_fields(N.PromptArgs, **{**fields, **kw})), None)

    for kw in ({"sequences": 2**24}, {"sequences": 2**23, "heads": 2, "kv_heads": 2}, {"sequences": 2**31 - 65},
               {"sequences": 2**31 - 20}, {"sequences": 1, "tokens": 2**30, "heads": 64, "kv_heads": 64}):
        assert status(**kw) == N.UNSUPPORTED, kw


def test_too_many_rows():
    lib = N.load_library()
    heads = dict(q=4096, k=4096, q_out=4096, k_out=4096, dtype=N.DTYPE_BF16, heads=4, kv_heads=2, dim=16,
                 normed=1, pairs=8, positions=4096, positions_dtype=N.DTYPE_I64, inv_freq=4096)
    for tokens in (2**32, 2**33, 2**40):
        args = N.pack_norm_rotary(*_fields(N.NormRotaryArgs, **heads, tokens=tokens))
        assert lib.omni_norm_rotary(args, None) == N.UNSUPPORTED
    read = dict(slots=4096, slots_dtype=N.DTYPE_I64, slots_stride=1, k=4096, v=4096, dtype=N.DTYPE_BF16)
    for tokens in (2**31, 2**33, 2**40):
        args = N.pack_read_cache(*_fields(N.ReadCacheArgs, **read, tokens=tokens, cache=_cache()))
        assert lib.omni_read_cache(args, None) == N.UNSUPPORTED
    paged = dict(q=4096, out=4096, dtype=N.DTYPE_BF16, table=4096, table_stride=4, table_columns=400,
                 lengths=4096, lengths_dtype=N.DTYPE_I32, max_length=3200, workspace=4096,
                 workspace_bytes=2**62)
    for batch, count in ((2**15, 2**9), (65535, 1024)):
        args = N.pack_paged(*_fields(N.PagedArgs, **paged, batch=batch, heads=count, cache=_cache()))
        assert lib.omni_paged_attention(args, None) == N.UNSUPPORTED
