"""The argument structs of the attention and cache operators, without a GPU: field for field the
header's, and refusals before any launch."""

from __future__ import annotations

import pytest
import torch

from sglang_omni_amd import _native as N
from tests.test_operator_abi import _header_fields

STRUCTS = [("omni_kv_cache", N.KvCacheStruct, N.pack_kv_cache),
           ("omni_norm_rotary_args", N.NormRotaryArgs, N.pack_norm_rotary),
           ("omni_read_cache_args", N.ReadCacheArgs, N.pack_read_cache),
           ("omni_prompt_args", N.PromptArgs, N.pack_prompt),
           ("omni_paged_args", N.PagedArgs, N.pack_paged)]


@pytest.mark.parametrize("name,args,pack", STRUCTS)
def test_fields_mirror_the_header(name, args, pack):
    assert list(args._fields_) == _header_fields(name)
    values = [0.5 + i if t is N.ctypes.c_float else (1 << 40) + i if t is not N.ctypes.c_int else i
              for i, (_, t) in enumerate(args._fields_)]
    packed, struct = pack(*values), bytes(args(*values))
    assert struct[:len(packed)] == packed and len(struct) - len(packed) < 8


def _chunks(length, units):
    """The chunks of a sequence, by the kernel's rule."""
    if length <= 512:
        return 1
    size = 256 if length * units <= 64 * 256 else 512 if length * units <= 512 * 256 else 1024
    return -(-length // size)


@pytest.mark.parametrize("heads,kv", [(8, 8), (32, 8), (64, 32), (14, 2), (20, 1), (6, 3), (40, 1), (5, 5)])
def test_workspace_holds_the_parts_of_every_length(heads, kv):
    lib = N.load_library()
    units = min(kv * -(-heads // kv // 16), 8)
    edges = [0, 1, 256, 257, 512, 513, 64 * 256 // units, 64 * 256 // units + 1, 512 * 256 // units,
             512 * 256 // units + 1, 40000, 131072, 10 ** 6]
    for bound in edges:
        held = lib.omni_paged_workspace(3, heads, kv, 16, bound) // (3 * heads * 18 * 4)
        for length in edges:
            if length <= bound:
                assert _chunks(length, units) <= max(held, 1), (bound, length)
        assert (held == 0) == (bound <= 512)


def _fields(args, **values):
    return [values.get(name, 0.5 if t is N.ctypes.c_float else 0) for name, t in args._fields_]


def test_refused_before_any_launch():
    """The C entry points check their arguments before the GPU is asked for anything: every call here
    has one thing wrong, and pointers that no launch could have read."""
    lib = N.load_library()
    entries = {"omni_norm_rotary_args": lib.omni_norm_rotary,
               "omni_read_cache_args": lib.omni_read_cache, "omni_prompt_args": lib.omni_prompt_attention,
               "omni_paged_args": lib.omni_paged_attention}
    for name, args, pack in STRUCTS[1:]:
        assert entries[name](None, None) == N.INVALID_ARG
        assert entries[name](pack(*[0] * len(args._fields_)), None) == N.INVALID_ARG

    def cache(**kw):
        base = dict(keys=4096, values=4096, dtype=N.DTYPE_BF16, stride_page=256, stride_head=128,
                    stride_token=16, pages=4, page_size=8, kv_heads=2, dim=16)
        struct = N.KvCacheStruct(*_fields(N.KvCacheStruct, **{**base, **kw}))
        cache.kept = struct
        return N.ctypes.addressof(struct)

    prompt = dict(q=4096, q_stride_token=64, q_stride_head=16, k=4096, k_stride_token=64, k_stride_head=16,
                  v=4096, v_stride_token=64, v_stride_head=16, out=4096, out_stride_token=64,
                  out_stride_head=16, dtype=N.DTYPE_BF16, tokens=0, key_tokens=8, heads=4, kv_heads=2,
                  dim=16, starts=4096, key_starts=4096, starts_dtype=N.DTYPE_I32, sequences=1, causal=1)

    def prompt_status(**kw):
        return lib.omni_prompt_attention(N.pack_prompt(*_fields(N.PromptArgs, **{**prompt, **kw})), None)

    assert prompt_status() == N.OK  # no tokens: nothing is launched
    for kw in ({"dtype": N.DTYPE_F32}, {"heads": 3}, {"kv_heads": 0}, {"dim": 12}, {"dim": 0},
               {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")}, {"scale": float("inf")},
               {"starts_dtype": N.DTYPE_F32}, {"sequences": -1}, {"q_stride_token": 60},
               {"k_stride_head": 4}, {"tokens": -1}, {"tokens": 8, "q": 4104}, {"tokens": 8, "k": 0},
               {"tokens": 8, "starts": 0}, {"tokens": 8, "key_starts": 2}, {"tokens": 8, "out": 0}):
        assert prompt_status(**kw) == N.INVALID_ARG, kw
    for kw in ({"dim": 264}, {"k_stride_token": (1 << 23) + 8}, {"key_tokens": 1 << 31}):
        assert prompt_status(**kw) == N.UNSUPPORTED, kw

    paged = dict(q=4096, q_stride_row=64, q_stride_head=16, out=4096, out_stride_row=64, out_stride_head=16,
                 dtype=N.DTYPE_BF16, batch=0, heads=4, table=4096, table_stride=4, table_columns=4,
                 lengths=4096, lengths_dtype=N.DTYPE_I32, max_length=32)

    def paged_status(held=None, **kw):
        fields = {**paged, "cache": cache(**(held or {})), **kw}
        return lib.omni_paged_attention(N.pack_paged(*_fields(N.PagedArgs, **fields)), None)

    assert paged_status() == N.OK
    for held in ({"keys": 0}, {"keys": 4104}, {"dtype": N.DTYPE_F32}, {"dtype": N.DTYPE_F16}, {"pages": 0},
                 {"page_size": 0}, {"pages": 1 << 20, "page_size": 1 << 11}, {"stride_token": 20},
                 {"dtype": N.DTYPE_FP8_E4M3}, {"kv_heads": 3}, {"kv_heads": 0}, {"dim": 24}):
        assert paged_status(held) == N.INVALID_ARG, held
    for kw in ({"cache": 0}, {"dtype": N.DTYPE_F32}, {"scale": 0.0}, {"q_stride_head": 12},
               {"lengths_dtype": N.DTYPE_F32}, {"max_length": -1}, {"batch": -1}, {"batch": 2, "q": 0},
               {"batch": 2, "lengths": 4098}, {"batch": 2, "table": 0},
               {"batch": 2, "max_length": 513}, {"batch": 2, "max_length": 513, "workspace": 4096,
                                                 "workspace_bytes": 2 * 4 * 3 * 18 * 4 - 1}):
        assert paged_status(**kw) == N.INVALID_ARG, kw
    assert paged_status(batch=65536) == paged_status(max_length=2**31 - 1) == N.UNSUPPORTED

    heads = dict(q=4096, q_stride_token=64, q_stride_head=16, k=4096, k_stride_token=64, k_stride_head=16,
                 v=4096, q_out=4096, k_out=4096, dtype=N.DTYPE_BF16, tokens=8, heads=4, kv_heads=2, dim=16,
                 normed=1, pairs=8, positions=4096, positions_dtype=N.DTYPE_I64, inv_freq=4096, slots=4096,
                 slots_dtype=N.DTYPE_I64)

    def heads_status(held=None, **kw):
        fields = {**heads, "cache": cache(**held) if held is not None else 0, **kw}
        return lib.omni_norm_rotary(N.pack_norm_rotary(*_fields(N.NormRotaryArgs, **fields)), None)

    assert heads_status(tokens=0) == heads_status({}, tokens=0) == N.OK
    for kw in ({"q": 0}, {"q_out": 0}, {"k": 0}, {"k_out": 0}, {"q": 4097}, {"pairs": 9}, {"pairs": -1},
               {"heads": 0, "kv_heads": 0}, {"dtype": N.DTYPE_I32}, {"layout": 2}, {"positions": 4},
               {"positions_dtype": N.DTYPE_F32}, {"inv_freq": 4}, {"q_weight": 2}, {"tokens": -1}):
        assert heads_status(**kw) == N.INVALID_ARG, kw
    for kw in ({"v": 0}, {"slots": 0}, {"slots_dtype": N.DTYPE_F32}):
        assert heads_status({}, **kw) == N.INVALID_ARG, kw
    for held in ({"dim": 32}, {"kv_heads": 1}, {"keys": 4097}):
        assert heads_status(held) == N.INVALID_ARG, held
    assert heads_status(dim=514) == N.UNSUPPORTED

    read = dict(slots=4096, slots_dtype=N.DTYPE_I64, slots_stride=1, tokens=8, k=4096, k_stride_token=32,
                k_stride_head=16, v=4096, v_stride_token=32, v_stride_head=16, dtype=N.DTYPE_BF16)

    def read_status(held=None, **kw):
        fields = {**read, "cache": cache(**(held or {})), **kw}
        return lib.omni_read_cache(N.pack_read_cache(*_fields(N.ReadCacheArgs, **fields)), None)

    assert read_status(tokens=0) == N.OK
    for kw in ({"held": {"dim": 24}}, {"held": {"keys": 4104}}, {"slots": 4}, {"slots_dtype": N.DTYPE_F32},
               {"tokens": -1}, {"cache": 0}, {"k": 0}, {"k": 4097}, {"dtype": N.DTYPE_FP8_E4M3}):
        assert read_status(**kw) == N.INVALID_ARG, kw


def test_tensors_off_the_gpu_are_refused():
    from sglang_omni_amd.kernels import PagedKvCache, prompt_attention

    q = torch.zeros(4, 2, 16, dtype=torch.bfloat16)
    with pytest.raises(N.OmniCodecError):
        prompt_attention(q, q, q, torch.tensor([0, 4]))
    with pytest.raises(N.OmniCodecError):
        PagedKvCache(q[None], q[None])
