"""Registers of the built kernels, from the metadata of the library's own code
objects: what a plan's workgroups a CU count on."""
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "igllm_amd", "libigl_hip.so")
READELF = "/opt/rocm/llvm/bin/llvm-readelf"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(data):
    """The gfx950 code objects of the library's bundles."""
    for m in re.finditer(MAGIC, data):
        at = m.end()
        count, at = struct.unpack_from("<Q", data, at)[0], at + 8
        for _ in range(count if count < 64 else 0):
            offset, size, name = struct.unpack_from("<QQQ", data, at)
            triple, at = data[at + 24:at + 24 + name], at + 24 + name
            if triple.endswith(b"gfx950") and size:
                yield data[m.start() + offset:m.start() + offset + size]


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """Name to metadata numbers, of the attention over the 4-bit ring."""
    if not os.path.exists(LIB) or not os.path.exists(READELF):
        pytest.skip("no built library, or no llvm-readelf")
    out = {}
    for i, blob in enumerate(code_objects(open(LIB, "rb").read())):
        if b"attend4_step_kernel" not in blob:
            continue
        path = tmp_path_factory.mktemp("co") / f"{i}.co"
        path.write_bytes(blob)
        notes = subprocess.run([READELF, "--notes", str(path)], check=True, capture_output=True, text=True).stdout
        for part in re.split(r"\n  - ", notes):
            name = re.search(r"\.name: +(\S*attend4\S*)", part)
            if name:
                out[name.group(1)] = {k: int(v) for k, v in re.findall(r"\.(\w+): +(\d+)\n", part + "\n")}
    assert len(out) > 10
    return out


def test_two_workgroups_a_cu(kernels):
    """Step workgroups, a wave a SIMD, are cut for two a CU, and a tile's eight waves lie
    two a SIMD: 512 registers a SIMD lane, so 256 a kernel, and 160 KiB of LDS."""
    for name, k in kernels.items():
        if "attend4_step" in name or "attend4_tile" in name:
            assert k["vgpr_count"] <= 256, (name, k)
            assert k["private_segment_fixed_size"] <= 32, (name, k)  # a few words of 512-slot steps
        if "attend4_step" in name:
            assert 2 * k["group_segment_fixed_size"] <= 160 << 10, (name, k)
