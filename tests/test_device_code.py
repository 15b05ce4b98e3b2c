"""What the compiler does not see to in the built device code: instructions written as inline assembly."""
import os
import re
import struct
import subprocess

import pytest

import spconv_amd

LLVM = "/opt/rocm/llvm/bin"


def code_objects(tmp_path):
    """The gfx950 code objects in the library, as files."""
    fat = tmp_path / "fatbin"
    subprocess.run([f"{LLVM}/llvm-objcopy", f"--dump-section=.hip_fatbin={fat}", spconv_amd.LIB_PATH, str(tmp_path / "copy.so")],
                   check=True)
    data, magic, out = fat.read_bytes(), b"__CLANG_OFFLOAD_BUNDLE__", []
    for m in re.finditer(magic, data):
        at = m.end()
        count, = struct.unpack_from("<Q", data, at)
        at += 8
        for _ in range(count):
            offset, size, n = struct.unpack_from("<QQQ", data, at)
            name = data[at + 24:at + 24 + n]
            at += 24 + n
            if b"gfx950" in name and size:
                f = tmp_path / f"{len(out)}.co"
                f.write_bytes(data[m.start() + offset:m.start() + offset + size])
                out.append(f)
    return out


def test_lds_loads_wait_for_m0(tmp_path):
    """A load straight into LDS takes its address from M0. Behind a scalar write of M0 the hardware needs one wait state, which the
    compiler gives its own such loads (s_nop, or another instruction between), but not those of an asm block."""
    spconv_amd.load_library()
    if not os.path.exists(f"{LLVM}/llvm-objdump"):
        pytest.skip("no disassembler")
    loads, bad = 0, []
    for f in code_objects(tmp_path):
        text = subprocess.run([f"{LLVM}/llvm-objdump", "-d", "--mcpu=gfx950", "--no-show-raw-insn", str(f)], check=True,
                              capture_output=True, text=True).stdout
        kernel, before = "", ""
        for line in text.splitlines():
            head = re.match(r"[0-9a-f]+ <(.*)>:", line)
            if head:
                kernel, before = head.group(1), ""
                continue
            ins = line.split("//")[0].strip()
            if not ins:
                continue
            if re.match(r"(buffer|global|scratch)_load", ins) and re.search(r"\blds\b|_lds_", ins):
                loads += 1
                if re.match(r"s_\w+ m0,", before):
                    bad.append((kernel, before, ins))
            before = ins
    assert loads > 0
    assert not bad, (len(bad), sorted({k for k, _, _ in bad})[:8])
