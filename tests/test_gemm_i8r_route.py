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
