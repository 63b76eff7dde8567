"""How long the gfx950 code of the built library waits between a matrix instruction and its result's first use — TEST
INFRASTRUCTURE ONLY.  The hardware does not hold back an instruction that comes too early: it works on what the
registers held before.  The compiler puts the waits in, but where a branch stands between the two it may count along the
longer of two ways that meet again."""

from __future__ import annotations

import re
import struct
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
_MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
# Wait states until a result may be read, as compilers leave them in straight code: passes of four clocks, and four more (matrix
# units of 16 bits) or two (of 32).
_WAITS = {"v_mfma_f32_16x16x32_f16": 8, "v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x4_f32": 10}
_REG = re.compile(r"(?<![a-z_0-9])([va])(?:(\d+)(?!\d)|\[(\d+):(\d+)\])")


def code_objects(library: Path):
    """The gfx950 code objects of a library that hipcc linked."""
    data, at = library.read_bytes(), 0
    while (at := data.find(_MAGIC, at)) >= 0:
        p, (n,) = at + 32, struct.unpack_from("<Q", data, at + 24)
        for _ in range(n if n < 16 else 0):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            if b"gfx950" in data[p + 24:p + 24 + length] and size:
                yield data[at + offset:at + offset + size]
            p += 24 + length
        at += len(_MAGIC)


def listing(code: bytes) -> str:
    with tempfile.NamedTemporaryFile(suffix=".o") as f:
        f.write(code)
        f.flush()
        return subprocess.run([str(OBJDUMP), "-d", "--no-show-raw-insn", f.name], capture_output=True, text=True, check=True).stdout


def listings(library: Path):
    with ThreadPoolExecutor(8) as pool:
        yield from pool.map(listing, code_objects(library))


def _registers(text):
    out = set()
    for kind, one, low, high in _REG.findall(text):
        out.update((kind, i) for i in (range(int(low), int(high) + 1) if low else (int(one),)))
    return out


def functions(text):
    """(name, [(address, operation, operands)]) of a listing."""
    name, body = None, []
    for line in text.splitlines():
        if line.startswith("0") and line.endswith(">:"):
            if body:
                yield name, body
            name, body = line[line.index("<") + 1:-2], []
        elif line.startswith("\t") and "// " in line:
            what, where = line.split("// ", 1)
            op, _, args = what.strip().partition(" ")
            body.append((int(where.split(":")[0], 16), op, args.strip()))
    if body:
        yield name, body


def early(body):
    """(matrix instruction, use, wait states between) of results that some way through a function's code uses too early."""
    place = {address: i for i, (address, _, _) in enumerate(body)}

    def target(i):
        jump = int(body[i][2]) & 0xFFFF
        return place.get(body[i][0] + 4 + 4 * (jump - (jump & 0x8000) * 2))

    found = []
    for i, (_, op, args) in enumerate(body):
        if "mfma" not in op:
            continue
        result, need = _registers(args.split(",")[0]), _WAITS[op]
        least, ways = {}, [(i + 1, 0)]
        while ways:
            j, waited = ways.pop()
            while j is not None and j < len(body) and waited < need and least.get(j, need) > waited:
                least[j] = waited
                _, use, operands = body[j]
                first, _, rest = operands.partition(",")
                if "mfma" in use:
                    a, b = (_registers(x) for x in rest.split(", ")[:2])
                    if (a | b) & result:
                        found.append((f"{op} {args}", f"{use} {operands}", waited))
                        break
                    if _registers(first) >= result:  # summed further or made anew, in order
                        break
                elif _registers(operands) & result:
                    stores = use.startswith(("global_store", "buffer_store", "scratch_store", "ds_write"))
                    if waited < need - (not stores and not _registers(rest) & result):
                        found.append((f"{op} {args}", f"{use} {operands}", waited))
                    break
                waited += int(operands) + 1 if use == "s_nop" else 1
                if use == "s_endpgm":
                    break
                if use == "s_branch":
                    j = target(j)
                    continue
                if use.startswith("s_cbranch"):
                    ways.append((target(j), waited))
                j += 1
    return found
