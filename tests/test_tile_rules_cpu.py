"""CPU: the host rules of the matrix-product tiles (csrc/tile_pick.h), compiled by themselves."""
import ctypes as C
import pathlib
import shutil
import subprocess

import pytest

CSRC = pathlib.Path(__file__).resolve().parent.parent / "two-towers-overlords_amd" / "csrc"
SOURCE = """
#include "tile_pick.h"
extern "C" int pick(long long M, long long N, int dtype) { return ttm::pick_tile(M, N, 1, dtype); }
extern "C" int parts(int edge, int gn, long long columns) { return ttm::row_parts(edge, gn, columns); }
"""
TYPES = {"f32": 1, "bf16": 2, "f16": 3}


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("clang++") or "/opt/rocm/bin/amdclang++"
    d = tmp_path_factory.mktemp("rules")
    (d / "rules.cpp").write_text(SOURCE)
    subprocess.run([cxx, "-std=c++17", "-O1", "-shared", "-fPIC", f"-I{CSRC}", str(d / "rules.cpp"), "-o", str(d / "rules.so")], check=True)
    lib = C.CDLL(str(d / "rules.so"))
    lib.pick.argtypes, lib.parts.argtypes = [C.c_longlong, C.c_longlong, C.c_int], [C.c_int, C.c_int, C.c_longlong]
    return lib


@pytest.mark.parametrize("dtype", TYPES)
def test_every_part_that_a_target_entry_adds_was_written(rules, dtype):
    """A softmax-loss gradient tile of `edge` candidates has two waves of edge / 2; a wave that starts behind the padded
    candidates writes no part.  The parts that are added are exactly those that are written, and they cover every candidate."""
    odd = set()
    for N in (1, 5, 64, 203, 300, 512, 1024, 1499, 2048, 3700, 4096, 5200, 8192):
        for V in [*range(1, 700, 13), 1900, 2297, 3600, 3700, 3900, 3968, 4089, 5200, 5400, 7000, 10000, 16000, 17003, 30522, 33001, 65536]:
            edge = rules.pick(N, V, TYPES[dtype])
            gn, ldg = -(-V // edge), -(-V // 128) * 128
            written = [p for p in range(2 * gn) if p * (edge // 2) < ldg]
            parts = rules.parts(edge, gn, ldg)
            assert written == list(range(parts)) and parts * (edge // 2) >= V, (N, V, edge)
            assert parts <= 2 * ((ldg + 63) // 64)  # what the workspace holds
            if parts < 2 * gn:
                odd.add((N, V))
    if dtype != "f32":
        assert {(3700, 3700), (2048, 7000), (8192, 30522)} <= odd
