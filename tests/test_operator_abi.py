"""The argument structs of the transformer step's operators, without a GPU: field for field the
header's, and packed as bytes exactly as ctypes lays them out."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest

from sglang_omni_amd import _native as N

HEADER = Path(__file__).resolve().parents[1] / "include" / "omni_codec.h"

STRUCTS = [("omni_block_fp8_args", N.BlockFp8Args, N.pack_block_fp8),
           ("omni_gated_norm_args", N.GatedNormArgs, N.pack_gated_norm),
           ("omni_rotary_args", N.RotaryArgs, N.pack_rotary),
           ("omni_logits_args", N.LogitsArgs, N.pack_logits)]
C_TYPES = {"int": ctypes.c_int, "int64_t": ctypes.c_int64, "float": ctypes.c_float}


def _header_fields(name):
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    fields = []
    for decl in filter(None, (d.strip() for d in body.split(";"))):
        words = decl.replace("const ", "").split(None, 1)
        pointer = words[0].endswith("*")
        for part in words[1].split(","):
            part = part.strip()
            kind = ctypes.c_void_p if pointer or part.startswith("*") else C_TYPES[words[0]]
            fields.append((part.lstrip("*").strip(), kind))
    return fields


@pytest.mark.parametrize("name,args,pack", STRUCTS)
def test_fields_mirror_the_header(name, args, pack):
    assert list(args._fields_) == _header_fields(name)


@pytest.mark.parametrize("name,args,pack", STRUCTS)
def test_packed_bytes_are_the_struct(name, args, pack):
    values = [0.5 + i if t is ctypes.c_float else (1 << 40) + i if t is not ctypes.c_int else i
              for i, (_, t) in enumerate(args._fields_)]
    packed = pack(*values)
    struct = bytes(args(*values))
    assert struct[:len(packed)] == packed and len(struct) - len(packed) < 8


def test_constants_match_the_header():
    text = HEADER.read_text()
    for name, value in {"OMNI_BLOCK_FP8_FEW_ROWS": N.BLOCK_FP8_FEW_ROWS,
                        "OMNI_NORM_RMS": N.NORM_RMS, "OMNI_NORM_LAYER": N.NORM_LAYER,
                        "OMNI_GATE_NONE": N.GATE_NONE, "OMNI_GATE_SIGMOID": N.GATE_SIGMOID,
                        "OMNI_GATE_TANH": N.GATE_TANH, "OMNI_ROTARY_HALF": N.ROTARY_HALF,
                        "OMNI_ROTARY_INTERLEAVED": N.ROTARY_INTERLEAVED}.items():
        assert int(re.search(rf"\b{name}\s*=\s*(\d+)", text).group(1)) == value, name


def test_refused_before_any_launch():
    """The C entry points check their arguments before the GPU is asked for anything."""
    lib = N.load_library()
    zeros = {name: pack(*[0] * len(args._fields_)) for name, args, pack in STRUCTS}
    assert lib.omni_block_fp8_gemm(zeros["omni_block_fp8_args"], None) == N.INVALID_ARG
    assert lib.omni_gated_residual_norm(zeros["omni_gated_norm_args"], None) == N.INVALID_ARG
    assert lib.omni_rotary(zeros["omni_rotary_args"], None) == N.INVALID_ARG
    assert lib.omni_adjust_logits(zeros["omni_logits_args"], None) == N.INVALID_ARG
    assert lib.omni_block_quantize(None, 1, 8, 4, 8, None, 16, None, 1, None) == N.INVALID_ARG
    assert lib.omni_block_quantize(None, 1, 8, 0, 8, None, 16, None, 1, None) == N.OK
    for entry in (lib.omni_block_fp8_gemm, lib.omni_gated_residual_norm, lib.omni_rotary,
                  lib.omni_adjust_logits):
        assert entry(None, None) == N.INVALID_ARG
