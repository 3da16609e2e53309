"""The sizes of the layers' launches (neus2_amd/csrc/launch_rules.h), compiled with the host compiler: no GPU needed."""
import ctypes as C
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WRAPPERS = """
#include "launch_rules.h"
extern "C" uint64_t plan(uint32_t m, uint32_t n, uint32_t k, uint32_t* out) {
	const N2LinearPlan p = n2_linear_plan(m, n, k);
	out[0] = p.tile; out[1] = p.splits; out[2] = p.k_per_split;
	return n2_linear_partial_bytes(p, m, n);
}
extern "C" uint32_t xcd_order(uint32_t block, uint32_t blocks) { return n2_xcd_order(block, blocks); }
extern "C" void tile_order(uint32_t tile, uint32_t tiles_m, uint32_t tiles_n, uint32_t* out) { n2_tile_order(tile, tiles_m, tiles_n, out[0], out[1]); }
extern "C" uint32_t norm_forward_blocks(uint32_t rows, uint32_t per, uint32_t threads) { return n2_layer_norm_forward_blocks(rows, per, threads); }
extern "C" uint32_t norm_backward_blocks(uint32_t rows, uint32_t per, uint32_t threads) { return n2_layer_norm_backward_blocks(rows, per, threads); }
extern "C" uint32_t few_rows(uint32_t m) { return n2_linear_few_rows(m); }
extern "C" uint32_t streams(uint32_t m, uint32_t n, uint32_t k) { return n2_linear_streams(m, n, k); }
extern "C" uint32_t stream_blocks(uint32_t m, uint32_t lds) { return n2_linear_stream_blocks(m, lds); }
extern "C" uint32_t dz_streams(uint64_t rows, uint64_t in, uint64_t out) { return n2_linear_dz_streams(rows, in, out); }
extern "C" uint32_t sum_blocks(uint32_t rows, uint32_t width) { return n2_linear_sum_blocks(rows, width); }
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("rules")
    src, so = d / "rules.cpp", d / "rules.so"
    src.write_text(WRAPPERS)
    subprocess.run([os.environ.get("CXX", "g++"), "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", os.path.join(ROOT, "neus2_amd", "csrc"), str(src), "-o", str(so)],
                   check=True, timeout=60)
    lib = C.CDLL(str(so))
    lib.plan.restype = C.c_uint64
    return lib


def test_every_value_of_k_is_in_one_split(rules):
    rng = random.Random(1)
    shapes = [(1, 1, 1), (0, 5, 7), (5, 7, 0), (1, 65536, 65536), ((1 << 32) - 1, 16, 16), (65536, 65536, (1 << 32) - 1), (64, 64, (1 << 32) - 1)]
    shapes += [tuple(max(1, int(2 ** rng.uniform(0, top))) for top in (18, 12, 18)) for _ in range(3000)]
    out = (C.c_uint32 * 3)()
    for m, n, k in shapes:
        partial = rules.plan(m, n, k, out)
        tile, splits, per = out
        assert tile in (64, 128, 256) and splits >= 1
        if splits == 1:
            assert per == k and partial == 0
        else:
            assert per % 64 == 0 and (splits - 1) * per < k <= splits * per and partial == 4 * splits * m * n


def test_what_the_products_take_at_most_in_partial_sums(rules):
    """A workspace stays within a few times the operands and 600 tiles' sums."""
    rng = random.Random(2)
    out = (C.c_uint32 * 3)()
    for _ in range(3000):
        m, n, k = (max(1, int(2 ** rng.uniform(0, top))) for top in (17, 12, 17))
        assert rules.plan(m, n, k, out) <= 4 * 1024 * 64 * 64 + 4 * 512 * 128 * 128 + 4 * 256 * 256 * 256, (m, n, k)


@pytest.mark.parametrize("m,n", [(1, 1), (1, 9), (9, 1), (4, 4), (5, 3), (64, 8), (7, 33), (130, 2)])
def test_every_tile_comes_once(rules, m, n):
    out = (C.c_uint32 * 2)()
    seen = set()
    for block in range(m * n):
        tile = rules.xcd_order(block, m * n)
        assert tile < m * n
        rules.tile_order(tile, m, n, out)
        assert out[0] < m and out[1] < n
        seen.add((out[0], out[1]))
    assert len(seen) == m * n


def test_blocks_of_the_passes_over_rows(rules):
    for rows in (1, 3, 4, 255, 4097, 1 << 20, (1 << 32) - 1):
        for per, threads in ((32, 256), (4, 256), (1, 256), (1, 1024)):
            for blocks, most in ((rules.norm_forward_blocks(rows, per, threads), 2048), (rules.norm_backward_blocks(rows, per, threads), 1024)):
                assert 1 <= blocks <= most and (blocks - 1) * per < rows
        for width in (1, 64, 65, 256, 257, 4096, 65536):
            assert 1 <= rules.sum_blocks(rows, width) <= 1024
    assert rules.norm_forward_blocks(0, 4, 256) == rules.norm_backward_blocks(0, 4, 256) == 0 and rules.sum_blocks(0, 8) == 0


def test_ways_change_where_their_measurements_cross(rules):
    assert rules.few_rows(1) and rules.few_rows(16) and not rules.few_rows(17)
    assert rules.streams(49152, 256, 256) and rules.streams(1 << 31, 1, 1)
    assert not rules.streams(49151, 256, 256) and not rules.streams(1 << 20, 257, 256) and not rules.streams(1 << 20, 256, 257)
    rules.dz_streams.argtypes = [C.c_uint64] * 3
    assert rules.dz_streams(1 << 18, 256, 256) and rules.dz_streams((1 << 31) - 1, 65536, 65536)
    assert not rules.dz_streams(65536, 256, 256) and not rules.dz_streams(1, 65536, 65536) and not rules.dz_streams(0, 1, 1)
    for rows in (49152, 49153, 100000, (1 << 31) - 1):
        for lds in (4096, 32768, 65536, 65537, 131072):
            blocks = rules.stream_blocks(rows, lds)
            assert 1 <= blocks <= (256 if lds > 65536 else 512) and (blocks - 1) * 256 < rows
