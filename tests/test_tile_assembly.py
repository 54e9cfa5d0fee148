"""The int8 tile kernels as they were built: m0, which their copies to LDS write in
assembly that cannot say so, has no other user that a copy could come between."""
import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

from pulsar_amd import _lib

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
OBJDUMP = next((p for p in ("/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump")) if p and Path(p).exists()), None)


def code_objects(data):
    """The gfx950 code objects of the bundles in a library's bytes."""
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        entry = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, n = struct.unpack_from("<QQQ", data, entry)
            name = data[entry + 24:entry + 24 + n]
            if name.endswith(b"gfx950"):
                yield data[at + offset:at + offset + size]
            entry += 24 + n
        at = data.find(MAGIC, at + 1)


@pytest.mark.skipif(OBJDUMP is None or not _lib.LIB_PATH.exists(), reason="no disassembler, or the library is not built")
def test_m0_is_the_copies_alone(tmp_path):
    kernels = copies = 0
    for i, code in enumerate(code_objects(_lib.LIB_PATH.read_bytes())):
        if b"i8_tile_kernel" not in code:
            continue
        path = tmp_path / f"{i}.o"
        path.write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", str(path)], capture_output=True, text=True,
                              check=True).stdout
        inside, before = False, ["", ""]
        for line in text.splitlines():
            head = re.match(r"[0-9a-f]+ <(.*)>:$", line)
            if head:
                inside = "i8_tile_kernel" in head[1]
                kernels += inside
            line = line.split("//")[0].strip()
            if inside and line:
                if re.search(r"\blds\b", line):
                    assert line.startswith("buffer_load_dwordx4"), line
                    assert before[0].startswith("s_mov_b32 m0, ") and before[1] == "s_nop 0", (before, line)
                    copies += 1
                if re.search(r"\bm0\b", before[0]):
                    assert re.search(r"\blds\b", line), (before, line)
                before = [before[1], line]
    assert kernels >= 3 * 10 and copies >= 100
