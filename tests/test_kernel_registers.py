"""CPU tests of what the compiler made of the kernels that fill their registers: spills show in the library's metadata."""

from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

TOOLS = Path("/opt/rocm/llvm/bin")
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def _code_objects(path: Path, tmp: Path):
    """The device code of each source of the library, as files."""
    section = tmp / "fatbin"
    subprocess.run([TOOLS / "llvm-objcopy", f"--dump-section=.hip_fatbin={section}", path, tmp / "copy"], check=True,
                   capture_output=True)
    data, at, count = section.read_bytes(), 0, 0
    while (at := data.find(MAGIC, at)) >= 0:
        entries, = struct.unpack_from("<Q", data, at + len(MAGIC))
        place = at + len(MAGIC) + 8
        for _ in range(entries):
            offset, size, length = struct.unpack_from("<QQQ", data, place)
            target = data[place + 24:place + 24 + length]
            place += 24 + length
            if b"gfx950" in target and size:
                out = tmp / f"{count}.elf"
                out.write_bytes(data[at + offset:at + offset + size])
                count += 1
                yield out
        at += len(MAGIC)


@pytest.fixture(scope="module")
def kernels(ctmr, native_loaded, tmp_path_factory):
    """(vector registers spilled, scratch bytes a lane) of each kernel by its mangled name."""
    if not (TOOLS / "llvm-objcopy").exists() or not shutil.which("/opt/rocm/llvm/bin/llvm-readelf"):
        pytest.skip("needs ROCm's llvm-objcopy and llvm-readelf")
    found = {}
    for code in _code_objects(Path(ctmr._lib.LIB_PATH), tmp_path_factory.mktemp("code")):
        notes = subprocess.run([TOOLS / "llvm-readelf", "--notes", code], check=True, capture_output=True, text=True).stdout
        for block in notes.split("  - .agpr_count:")[1:]:
            get = lambda name: re.search(rf"\.{name}:\s*(\S+)", block).group(1)
            found[get("symbol")] = int(get("vgpr_spill_count")), int(get("private_segment_fixed_size"))
    return found


# element type, head width, cap (none, shifted, exact) -> registers that dq's kernel without a bias spilled when its waves a
# SIMD were chosen; all others spill none
DQ_SPILLS = {("DF16b", 32, 0): 3, ("DF16b", 32, 1): 7, ("DF16b", 32, 2): 9, ("DF16b", 64, 1): 5, ("DF16b", 64, 2): 12,
             ("DF16_", 32, 0): 2, ("DF16_", 32, 1): 7, ("DF16_", 32, 2): 15, ("DF16_", 64, 1): 5, ("DF16_", 64, 2): 13,
             ("DF16_", 128, 1): 2}


def test_gradients_without_a_bias_keep_their_registers(kernels):
    seen = 0
    for name, (spills, scratch) in kernels.items():
        m = re.search(r"attention_dq_kernelI(DF16b|DF16_|f)Li(\d+)ELNS0_3CapE(\d)ELi0E", name)
        if m is None:
            continue
        seen += 1
        most = DQ_SPILLS.get((m.group(1), int(m.group(2)), int(m.group(3))), 0)
        assert spills <= most and scratch <= 64, (name, spills, scratch)
    assert seen == 24
