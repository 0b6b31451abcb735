"""The registers of the built kernels, from the notes of the library's code objects: what decides how many waves share a SIMD, and
changes with the compiler's flags without any test of results seeing it."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from mi355q import _lib as L

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


def code_objects(data):
    """The gfx950 ELF images of every offload bundle in a host library."""
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + len(magic))
        p = at + len(magic) + 8
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + length]
            p += 24 + length
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(magic, at + 1)


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: (vector registers, spilled ones)}"""
    if not os.path.exists(READELF) or not shutil.which("c++filt"):
        pytest.skip("no ELF reader")
    found, path = {}, tmp_path_factory.mktemp("elf") / "x.co"
    with open(L.LIB_PATH, "rb") as f:
        data = f.read()
    for image in code_objects(data):
        path.write_bytes(image)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for m in re.finditer(r"\.name:\s+(_Z\S+).*?\.vgpr_count:\s+(\d+).*?\.vgpr_spill_count:\s+(\d+)", notes, re.S):
            found[m.group(1)] = (int(m.group(2)), int(m.group(3)))
    assert found
    return found


@pytest.mark.parametrize("pattern,least", [
    (r"decode_attn_gqa_kernelINS_\d+b?f16_tELi[12]E", 12),  # 8-bit caches
    (r"tree_attn_kernelINS_\d+b?f16_tELi[012]ELi(64|128)E", 48)])
def test_two_waves_share_a_simd(kernels, pattern, least):
    # 512 registers a SIMD lane: at most 256 a wave, none in memory
    mine = {k: v for k, v in kernels.items() if re.search(pattern, k)}
    assert len(mine) >= least
    assert not {k: v for k, v in mine.items() if v[0] > 256 or v[1] > 0}
