"""What the compiler gave the kernels: read from the built library's own code objects (no GPU needed)."""
import os
import re
import subprocess

import pytest

READELF = "/opt/rocm/llvm/bin/llvm-readelf"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: {metadata field: number}} of the library's gfx950 code objects"""
    from aniportrait_amd import _lib as L
    if not os.path.exists(READELF):
        pytest.skip("no llvm-readelf")
    data = open(L.LIB_PATH, "rb").read()
    starts = [m.start() for m in re.finditer(b"\x7fELF\x02\x01\x01\x40", data)]   # ELF64, little-endian, AMDGPU HSA
    assert starts
    got = {}
    for a, b in zip(starts, starts[1:] + [len(data)]):
        f = tmp_path_factory.mktemp("co") / "code.o"
        f.write_bytes(data[a:b])
        notes = subprocess.run([READELF, "--notes", str(f)], capture_output=True, text=True).stdout
        for part in re.split(r"\n  - \.a", notes)[1:]:                            # (each kernel's map begins with .agpr_count)
            name = re.search(r"\.name:\s+(\S+)", part[part.rindex(".max_flat_workgroup_size"):] if ".max_flat_workgroup_size" in part else part)
            got[name[1]] = {k: int(v) for k, v in re.findall(r"\.(private_segment_fixed_size|vgpr_spill_count|vgpr_count):\s+(\d+)", part)}
    return got


def test_learned_attention_keeps_its_registers(kernels):
    """no vector register of the attention with learned positions goes to scratch: the reloads would wait for the tiles' DMA"""
    mine = {n: k for n, k in kernels.items() if "mapattn" in n or "head_norm" in n}
    assert len(mine) > 80, sorted(kernels)[:5]
    spilled = {n: k["vgpr_spill_count"] for n, k in mine.items() if k["vgpr_spill_count"]}
    assert not spilled, spilled
