"""Which kernel the int8 row product takes (gemm_i8r_route.h), compiled for the
CPU: the few-token kernel up to 16 tokens, each tile somewhere, larger tiles
only where there are enough of them, and a choice at every size."""

import ctypes
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "gemm_i8r_route.h"
extern "C" int route(int64_t n, int64_t rows, int64_t cols) { return dnx::i8r_route(n, rows, cols); }
"""


def compiled_route(folder):
    (folder / "r.cpp").write_text(SOURCE)
    so = str(folder / "r.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so, str(folder / "r.cpp"),
                    "-I", os.path.join(ROOT, "dianoia_amd", "csrc")], check=True)
    f = ctypes.CDLL(so).route
    f.argtypes, f.restype = [ctypes.c_int64] * 3, ctypes.c_int
    return f


@pytest.fixture(scope="module")
def route(tmp_path_factory):
    return compiled_route(tmp_path_factory.mktemp("route"))


# A shape of odd sizes for each tile kernel, in the order of its table.
SHAPES = [(17, 520, 4096), (63, 4300, 2048), (127, 4100, 2048), (255, 4099, 2080),
          (511, 4098, 4096), (1023, 6145, 1056), (2047, 8189, 1184)]
MORE = [(2047, 2049, 4096), (1023, 8193, 1056)]


def test_each_kernel_is_taken(route):
    assert [route(*s) for s in SHAPES] == list(range(7))
    assert all(route(n, 4096, 2048) == -1 for n in (1, 2, 15, 16))
    assert route(17, 4096, 2048) >= 0


def test_every_size_has_one(route):
    for n in (17, 64, 1000, 1 << 22):
        for rows in (1, 33, 5000, 1 << 30):
            for cols in (32, 1120, 131040):
                assert 0 <= route(n, rows, cols) < 7


FEW = """
#include "gemm_i8r_route.h"
extern "C" int few(int64_t n, int64_t rows) { return dnx::i8r_few_tiles(n, rows); }
"""


def test_few_tokens_tiles_of_a_workgroup(tmp_path):
    """Two tiles of rows a workgroup from five tokens on, where they leave no CU
    more rows than one would, or where there are very many rows."""
    (tmp_path / "f.cpp").write_text(FEW)
    so = str(tmp_path / "f.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so, str(tmp_path / "f.cpp"),
                    "-I", os.path.join(ROOT, "dianoia_amd", "csrc")], check=True)
    few = ctypes.CDLL(so).few
    few.argtypes, few.restype = [ctypes.c_int64] * 2, ctypes.c_int
    for n in (1, 4):
        assert all(few(n, rows) == 1 for rows in (1, 6144, 8192, 32769, 1 << 21))
    for n in (5, 16):
        # 256 CUs: one round of 16 or 32 rows a workgroup up to 4096 and 8192 rows.
        for rows, tiles in ((1, 1), (4096, 1), (4097, 2), (6144, 2), (8192, 2), (8193, 1), (12288, 1),
                            (12289, 2), (16384, 2), (20480, 1), (32768, 2), (32769, 2), (36864, 2),
                            (128256, 2)):
            assert few(n, rows) == tiles, (n, rows)
