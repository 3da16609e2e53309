"""Registers and waves per SIMD of kernels whose times depend on them, as the compiler reports them: no GPU needed."""
import os
import re
import subprocess

import pytest

from neus2_amd import build


def resources(source, directory):
    """The kernels of a source: mangled name -> (waves per SIMD, vector registers, spilled ones)."""
    out = subprocess.run([build.HIPCC, *build.FLAGS, "--cuda-device-only", "-Rpass-analysis=kernel-resource-usage", "-c", os.path.join(build.CSRC, source), "-o", str(directory / "device.o")],
                         capture_output=True, text=True, check=True, timeout=300).stderr
    found = {}
    for part in out.split("Function Name: ")[1:]:
        waves, registers, spilled = (int(re.search(what + r": (\d+)", part)[1]) for what in (r"Occupancy \[waves/SIMD\]", r"\bVGPRs", "VGPRs Spill"))
        found[part.split()[0]] = waves, registers, spilled
    return found


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc")
def test_the_lattices_fine_levels_have_their_waves(tmp_path):
    """One branch with more registers takes waves from all of them: six per SIMD fit 80, and what small launches have on purpose is five."""
    found = {k: v for k, v in resources("lattice.hip", tmp_path).items() if "lattice_fine_kernel" in k}
    assert sorted(v[0] for v in found.values()) == [5, 6]
    assert all(registers <= 80 and spilled == 0 for _, registers, spilled in found.values())


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc")
def test_the_linear_layers_sums_stay_in_registers(tmp_path):
    """A product's tile is most of a wave's registers: a spilled one goes to memory in every stage."""
    found = resources("linear.hip", tmp_path)
    assert sum("product_kernel" in k for k in found) >= 36 and sum("stream_" in k for k in found) >= 54
    assert not [k for k, v in found.items() if v[2] != 0]


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="needs hipcc")
def test_the_norms_kernels_are_those_that_rows_can_reach(tmp_path):
    """Rows end at 16 384 values: 1024 lanes take them in two vectors of eight, or four of four."""
    found = {k: v for k, v in resources("layer_norm.hip", tmp_path).items() if "layer_norm_" in k}
    assert len(found) == 2 * (4 * 9 + 10)
    assert sorted("ffLj1024ELj4E" in k for k in found if "Lj4E" in k) == [True, True]
    # a row stays in its lanes' registers, the widest too
    assert not {k: v for k, v in found.items() if v[2] != 0}
