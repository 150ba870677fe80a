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


@pytest.mark.parametrize("name,maps", [("void mapattn_rows_kernel<2>(MapAttnArgs, float)", 2), ("_Z19mapattn_rows_kernelILi2EEv11MapAttnArgsf", 2),
                                       ("void mapattn_rows_kernel<1>(MapAttnArgs, float)", 1), ("_Z19mapattn_rows_kernelILi1EEv11MapAttnArgsf", 1),
                                       ("_Z17mapattn_dq_kernelIDF16bLi2ELi8ELi8ELi32ELi4ELi1EEv11MapAttnArgs", 2),
                                       ("_Z17mapattn_dq_kernelIDF16_Li1ELi4ELi2ELi64ELi4ELi2EEv11MapAttnArgs", 1)])
def test_counter_summaries_tell_one_map_from_two(name, maps):
    import importlib.util
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tools", "pmc_summarize.py")
    spec = importlib.util.spec_from_file_location("pmc_summarize", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    assert mod.family(name) == ("relative_attention_kernels", "differential_attention_kernels")[maps - 1]
