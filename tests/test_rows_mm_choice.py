"""The kernel that the float products choose, without a GPU: the choice is compiled for the host."""
if __name__ == "__main__":  # `python tests/<file>.py`, as the reference runs its tests
    import sys as _sys

    import pytest as _pytest
    _sys.exit(_pytest.main([__file__, "-q"]))
import ctypes
import subprocess
from pathlib import Path

import pytest

import _rows_paths as P
from jjjetson_ops_amd import build, capi

CODES = {"f32": capi.DTYPE_F32, "f16": capi.DTYPE_F16, "bf16": capi.DTYPE_BF16}
CHOICE = """
#include "rows_mm.hpp"
extern "C" void choice(int mode, int dtype, int P, int Q, int K, int halves, int n_experts, int *out) {
    const auto c = jjo::rows_mm_choose((jjo::RowsMode)mode, dtype, P, Q, K, halves, n_experts);
    out[0] = c.tile == jjo::kRowsDirect ? 0 : c.tile == jjo::kRowsTile64 ? 64 : c.tile == jjo::kRowsTile128 ? 128
             : c.tile == jjo::kRowsTile160 ? 160 : 256;
    out[1] = c.slices;
}
"""


@pytest.fixture(scope="module")
def choose(tmp_path_factory):
    if not Path(build.HIPCC).exists():
        pytest.skip("no hipcc")
    at = tmp_path_factory.mktemp("choice")
    (at / "choice.hip").write_text(CHOICE)
    subprocess.run([build.HIPCC, *build.HIP_FLAGS, "--offload-host-only", "-O1", "-shared", str(at / "choice.hip"),
                    str(build.CSRC / "rows_choose.hip"), "-o", str(at / "choice.so")], check=True, capture_output=True)
    lib = ctypes.CDLL(str(at / "choice.so"))

    def call(mode, name, cols, rows, sums, halves=1, experts=0):
        out = (ctypes.c_int * 2)()
        lib.choice(mode, CODES[name], cols, rows, sums, halves, experts, out)
        return out[0], out[1]
    return call


def _is(got, tile, slices):
    assert got[0] == tile and (got[1] > 1 if slices == 0 else got[1] == slices), (got, tile, slices)


def test_sizes_reach_their_kernels(choose):
    for (name, k, n, t), tile, slices in P.LINEAR:
        _is(choose(P.FORWARD, name, n, t, k), tile, slices)
    for (name, k, n, t), tile, slices in P.WEIGHTS:
        _is(choose(P.WEIGHT, name, k, n, t), tile, slices)
    for (name, h, i, counts), tile, slices in P.SWIGLU_FORWARD:
        _is(choose(P.SWIGLU, name, i, sum(counts), h, experts=len(counts)), tile, slices)
    for (name, h, i, counts), tile, slices in P.SWIGLU_WEIGHTS:
        _is(choose(P.WEIGHT, name, h, i, sum(counts), 2, len(counts)), tile, slices)


def _workgroups(got, cols, rows):
    return -(-cols // got[0]) * -(-rows // got[0]) * got[1]


@pytest.mark.parametrize("name", list(CODES))
def test_rows_without_alignment_get_kernels_that_run(choose, name):
    """Sizes that are no multiples of 16 bytes: tiles of 64 or 128, and slices that fill the CUs with those; never the
    large tiles, and of 16 bits never the direct kernel."""
    piece = 4 if name == "f32" else 8
    for rows in (1, 7, 16, 40, 64, 128, 256, 512, 2047):
        for cols, sums in ((4096, 4095), (4095, 4095), (1408, 2047), (11008, 4094)):
            got = choose(P.FORWARD, name, cols, rows, sums)
            assert got[0] in ((0, 64, 128) if name == "f32" and rows <= 16 else (64, 128)), (rows, cols, sums, got)
            if got[0] and sums > 32 * piece * 8:
                assert _workgroups(got, cols, rows) >= 128, (rows, cols, sums, got)
            got = choose(P.INPUT, name, sums, rows, cols)
            assert got[0] in (64, 128) and _workgroups(got, sums, rows) >= 64, (rows, cols, sums, got)
            assert choose(P.WEIGHT, name, sums, cols, rows)[0] in (64, 128)
            assert choose(P.SWIGLU, name, cols, rows * 8, sums, experts=8)[0] in ((0, 64, 128) if name == "f32" else (64, 128))
    # K aligned, the output's columns not: the tiles of 160 and 256 rows write whole groups of eight columns
    assert choose(P.FORWARD, name, 14337, 2047, 4096)[0] in (64, 128)
    # less than a piece: tiles of 128, which these run on
    if name != "f32":
        assert choose(P.FORWARD, name, 4096, 2047, 7)[0] == 128 and choose(P.WEIGHT, name, 4096, 5, 2047)[0] == 128


def test_few_rows_of_experts(choose):
    """fp32 on the direct kernel at any size (a tile's products would cost what 64 rows do); 16 bits where the tiles are
    fewer than the CUs."""
    for cols, sums, experts in ((4096, 512, 8), (4096, 2048, 8), (1408, 2048, 64), (704, 4096, 16)):
        for rows in (1, 8, 32, 8 * experts):
            if rows <= 8 * min(experts, rows):
                assert choose(P.FORWARD, "f32", cols, rows, sums, experts=experts)[0] == 0, (cols, sums, rows)
                assert choose(P.SWIGLU, "f32", cols, rows, sums, experts=experts)[0] == 0, (cols, sums, rows)
    for name in ("f16", "bf16"):
        assert choose(P.FORWARD, name, 1408, 8, 2048, experts=64)[0] == 0
        assert choose(P.FORWARD, name, 4096, 8, 2048, experts=8)[0] == 64
        assert choose(P.FORWARD, name, 4096, 8, 14336, experts=8)[0] == 0
        assert choose(P.SWIGLU, name, 1408, 8, 2048, experts=64)[0] == 64
