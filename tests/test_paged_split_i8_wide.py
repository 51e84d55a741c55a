"""Where the attention over int8 caches takes blocks of 64 rows (paged_split.h), compiled
for the CPU: as measured, and in the shapes that test_gpu_paged_i8_wide.py runs."""

import ctypes
import os
import subprocess

import pytest

from test_gpu_paged_i8_wide import BOUNDED, OWN, PREFIX

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "paged_split.h"
extern "C" int kinds(int64_t seqs, int64_t tokens, int64_t max_tokens, int64_t group,
                     int64_t kv_heads, int64_t prefix, int64_t len, int64_t hd) {
  const dnx::PagedSplit s =
      dnx::paged_split(seqs, tokens, max_tokens, group, kv_heads, prefix, len, false, (int)hd);
  return (s.own.wide ? 1 : 0) + (s.prefix.runs > 0 && s.prefix.wide ? 2 : 0) + (s.joined > 0 ? 4 : 0);
}
"""


@pytest.fixture(scope="module")
def kinds(tmp_path_factory):
    d = tmp_path_factory.mktemp("kinds")
    (d / "s.cpp").write_text(SOURCE)
    so = str(d / "s.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so, str(d / "s.cpp"),
                    "-I", os.path.join(ROOT, "dianoia_amd", "csrc")], check=True)
    f = ctypes.CDLL(so).kinds
    f.argtypes = [ctypes.c_int64] * 8
    return f


@pytest.mark.parametrize("seqs,each,heads,kv,prefix,keys,hd,own,shared", [
    (1, 64, 32, 8, 0, 256, 128, False, False), (1, 512, 32, 8, 0, 2048, 128, False, False),
    (1, 2048, 32, 8, 0, 2048, 128, False, False), (16, 256, 32, 8, 0, 256, 128, True, False),
    (64, 64, 32, 8, 0, 64, 128, True, False), (64, 64, 32, 8, 0, 1024, 128, True, False),
    (1, 1024, 12, 4, 0, 16384, 64, False, False), (16, 64, 12, 4, 0, 64, 64, True, False),
    (256, 1, 32, 8, 1000, 60, 128, False, False), (512, 1, 8, 1, 16384, 60, 128, False, True),
    (128, 1, 8, 1, 16384, 60, 128, False, True), (64, 1, 8, 1, 16384, 60, 128, False, False),
    (8, 4, 32, 8, 0, 10000, 128, False, False), (1, 1, 32, 8, 100000, 60, 128, False, False)])
def test_measured_shapes(kinds, seqs, each, heads, kv, prefix, keys, hd, own, shared):
    assert kinds(seqs, seqs * each, each, heads // kv, kv, prefix, keys, hd) & 3 == own + 2 * shared


def test_shapes_of_the_gpu_tests(kinds):
    for i, (counts, lens, prefix, heads, kv, _) in enumerate(OWN + PREFIX):
        for hd in (64, 128):
            kind = kinds(len(counts), sum(counts), max(counts), heads // kv, kv, prefix, max(lens), hd)
            assert kind & (1 if i < len(OWN) else 2) and kind < 4, (i, kind)
    assert kinds(len(BOUNDED[0]), sum(BOUNDED[0]) + 3, 700, 2, 8, 0, 190, 64) == 1


def test_bounds_of_sequences_do_not_count_as_rows(kinds):
    """Up to 20 new tokens of each of 64 sequences, 83 in all."""
    assert kinds(64, 83, 20, 4, 2, 0, 200, 128) == 0
    assert kinds(64, 64 * 20, 20, 4, 8, 0, 200, 128) == 1
