"""Launches of products beyond what one launch has threads for (neus2_amd/csrc/launch_rules.h), compiled with the host compiler: no GPU needed."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WRAPPERS = """
#include "launch_rules.h"
extern "C" void plan(uint32_t m, uint32_t n, uint32_t k, uint32_t* out) {
	const N2LinearPlan p = n2_linear_plan(m, n, k);
	out[0] = p.tile; out[1] = p.splits; out[2] = p.k_per_split;
}
extern "C" uint32_t launch_rows(uint32_t m, uint32_t tile, uint32_t tiles_n, uint32_t splits) { return n2_linear_launch_rows(m, tile, tiles_n, splits); }
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text(WRAPPERS)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "neus2_amd", "csrc"), str(src), "-o", str(so)],
                   check=True, timeout=60)
    return C.CDLL(str(so))


def test_a_products_launches_have_threads_for_their_rows(rules):
    """The threads of a launch are counted in 32 bits; what is more comes in several, each of whole tiles."""
    out = (C.c_uint32 * 3)()
    rng = random.Random(3)
    shapes = [((1 << 31) - 1, 1, 1), ((1 << 31) - 1, 65, 8), ((1 << 31) - 1, 65536, 65536), (1 << 30, 16, 3), (110_000_000, 257, 257), (1, 1, 1), (300, 2048, 2048)]
    shapes += [tuple(max(1, int(2 ** rng.uniform(0, top))) for top in (31, 16, 16)) for _ in range(3000)]
    cut = 0
    for m, n, k in shapes:
        rules.plan(m, n, k, out)
        tile, splits, _ = out
        threads, tiles_n = 512 if tile == 256 else 256, -(-n // tile)
        rows = rules.launch_rows(m, tile, tiles_n, splits)
        assert 1 <= rows <= m and (rows == m or (rows % tile == 0 and splits == 1)), (m, n, k)
        assert -(-rows // tile) * tiles_n * splits * threads < 1 << 32, (m, n, k)
        cut += rows < m
    assert cut >= 4
    # a product whose rows are widths is never cut
    for k in (1, 300, 1 << 18, (1 << 31) - 1):
        for m in (1, 257, 65536):
            for n in (1, 257, 65536):
                rules.plan(m, n, k, out)
                tile, splits, _ = out
                assert rules.launch_rows(m, tile, -(-n // tile), splits) == m
