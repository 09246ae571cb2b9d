"""The wait states of the built library's matrix products, without a GPU: along every path from a product
no other instruction touches its result, and along every path from a scalar register that a vector
instruction has written no memory instruction takes it as an operand, before the hardware has it there.

The compiler counts these states itself, but where paths meet right after a product it counts along one of
them alone, and a kernel has to add what is missing; which places those are changes with any change of the
code around them."""

from __future__ import annotations

import functools
import re
import shutil
import struct
import subprocess
from concurrent.futures import ProcessPoolExecutor
from pathlib import Path

import pytest

from sglang_omni_amd import _native as N

OBJDUMP = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin") or shutil.which("llvm-objdump")

# Until another instruction may use a product's result: its passes (8, for 16 x 16 x 32 4) and four more; for the
# float32 one, which the fast cores do not take, two more.
PRODUCTS = {"32x32x16_": 12, "16x16x32_": 8, "16x16x128_": 12, "16x16x4_f32": 10}
SCALARS = 5  # until a memory instruction may take a scalar register that a vector instruction wrote


def code_objects(library: bytes):
    """The gfx950 code objects bundled in a library."""
    at = library.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        count, = struct.unpack_from("<Q", library, at + 24)
        entry = at + 32
        for _ in range(count):
            offset, size, name = struct.unpack_from("<QQQ", library, entry)
            target = library[entry + 24:entry + 24 + name]
            entry += 24 + name
            if b"gfx950" in target and size:
                yield library[at + offset:at + offset + size]
        at = library.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 24)


def kernels(listing: str):
    """(name, [(operation, operands, address, branch target or None)]) of a disassembly."""
    name, code, base = None, [], 0
    for line in listing.splitlines():
        if line.startswith("\t") and name:
            text, _, rest = line.partition("// ")
            if not rest:  # padding
                continue
            operation, _, operands = text.strip().partition(" ")
            target = None
            if operation.startswith(("s_branch", "s_cbranch")):
                offset = re.search(r"<[^>]*?(?:\+0x([0-9a-f]+))?>", rest)
                target = base + int(offset[1] or "0", 16)
            code.append((operation, operands.strip(), int(rest.partition(":")[0], 16), target))
        elif line.endswith(">:"):
            if code:
                yield name, code
            address, _, label = line[:-2].partition(" <")
            name, code, base = label, [], int(address, 16)
    if code:
        yield name, code


@functools.lru_cache(maxsize=None)
def registers(operands: str) -> tuple[frozenset, ...]:
    """The registers of each operand."""
    out = []
    for operand in re.split(r",\s*", operands):
        m = re.match(r"-?\|?([vas])(?:\[(\d+):(\d+)\]|(\d+))(?!\w)", operand)
        if m is None:
            out.append(frozenset())
        else:
            first = int(m[2] or m[4])
            out.append(frozenset((m[1], i) for i in range(first, int(m[3] or m[4]) + 1)))
    return tuple(out)


def touched(operation: str, operands: str) -> frozenset:
    """What an instruction must not touch of a running product's result. Another product that goes on from it
    gets it in time by itself."""
    parts = registers(operands)
    if operation.startswith("v_mfma"):
        return parts[1] | parts[2]
    if operation.startswith(("v_", "ds_", "buffer_", "global_", "scratch_", "flat_")):
        return frozenset().union(*parts)
    return frozenset()


def faults(code) -> list[str]:
    """Uses that come too early on some path."""
    at = {address: i for i, (_, _, address, _) in enumerate(code)}
    found = []

    def walk(start, states, early, written):
        paths, best = [(start + 1, 0)], {}
        while paths:
            i, waited = paths.pop()
            if waited >= states or i >= len(code) or best.get(i, states) <= waited:
                continue
            best[i] = waited
            operation, operands, _, target = code[i]
            if early(operation, operands):
                found.append(f"{waited} of {states} states after {' '.join(code[start][:2])}: "
                             f"{operation} {operands}")
                return
            if operation.startswith(("s_endpgm", "s_setpc")) or written(operation, operands):
                continue
            waited += int(operands, 0) + 1 if operation == "s_nop" else 1
            if target is not None:
                paths.append((at[target], waited))
            if operation != "s_branch":
                paths.append((i + 1, waited))

    for i, (operation, operands, _, _) in enumerate(code):
        if operation.startswith("v_mfma"):
            states = next(n for kind, n in PRODUCTS.items() if kind in operation)
            result = registers(operands)[0]
            walk(i, states, lambda o, x: not result.isdisjoint(touched(o, x)), lambda o, x: False)
        elif operation.startswith(("v_readfirstlane", "v_readlane")):
            scalar = registers(operands)[0]
            walk(i, SCALARS,
                 lambda o, x: o.startswith(("buffer_", "global_", "scratch_", "flat_"))
                 and not scalar.isdisjoint(frozenset().union(*registers(x))),
                 lambda o, x: o.startswith("s_") and o not in ("s_nop", "s_waitcnt")
                 and registers(x)[0] == scalar)
    return found


def listed(*lines: str):
    """A disassembly of lines of code, at 8 bytes each; <n> is a branch to line n."""
    text = ["0000000000001000 <k>:"]
    for i, line in enumerate(lines):
        line = re.sub(r"<(\d+)>", lambda m: f"<k+0x{8 * int(m[1]):x}>", line)
        code, _, target = line.partition(" <")
        text.append(f"\t{code} // {0x1000 + 8 * i:012X}: BF800000" + (f" <{target}" if target else ""))
    (_, code), = kernels("\n".join(text))
    return code


def test_the_walk_sees_a_use_on_the_shorter_way():
    product = "v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], v[0:15]"
    use = "v_mov_b32_e32 v40, v14"
    assert faults(listed(product, "s_nop 10", use, "s_endpgm"))
    assert not faults(listed(product, "s_nop 11", use, "s_endpgm"))
    # straight on two states, around twelve: a count along the longer way alone sees nothing
    around = (product, "s_cbranch_scc0 4 <4>", "s_nop 9", "s_nop 0", use, "s_endpgm")
    assert faults(listed(*around)) == [f"1 of 12 states after {product}: {use}"]
    # a loop's way back; a result that the next product goes on from
    assert faults(listed(use, product, "s_cbranch_scc1 0 <0>", "s_endpgm"))
    assert not faults(listed(product, product, "s_nop 15", use, "s_endpgm"))
    scalar = "v_readfirstlane_b32 s5, v1"
    load = "buffer_load_dwordx4 v2, s[4:7], 0 offen lds"
    assert faults(listed(scalar, "s_nop 3", load, "s_endpgm"))
    assert not faults(listed(scalar, "s_nop 4", load, "s_endpgm"))
    assert not faults(listed(scalar, "s_mov_b32 s5, 0", load, "s_endpgm"))


def examined(path: Path) -> tuple[int, list[str]]:
    """The products of a code object, and the faults of its kernels."""
    products, bad, listing = 0, [], path.with_suffix(".txt")
    with open(listing, "w") as out:
        subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(path)], check=True, stdout=out)
    for name, code in kernels(listing.read_text()):
        products += sum(operation.startswith("v_mfma") for operation, *_ in code)
        bad += [f"{name}: {fault}" for fault in faults(code)]
    return products, bad


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
@pytest.mark.skipif(not N.LIB_PATH.exists(), reason="the library is not built")
def test_every_kernel_of_the_library(tmp_path):
    paths = []
    for i, blob in enumerate(code_objects(N.LIB_PATH.read_bytes())):
        paths.append(tmp_path / f"{i}.co")
        paths[-1].write_bytes(blob)
    with ProcessPoolExecutor(4) as pool:
        results = list(pool.map(examined, paths))
    assert sum(products for products, _ in results) > 10000
    bad = [fault for _, faults_of in results for fault in faults_of]
    assert not bad, bad[:5]
