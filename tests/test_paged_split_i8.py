"""How the attention over int8 caches deals its rows and keys (paged_split.h),
compiled for the CPU as the workgroups do it: every block of rows of every run
and key head has one workgroup, in whole rounds of the XCDs, and the heads of a
run that go to one XCD really do."""

import ctypes
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "paged_split.h"
extern "C" void split_of(int64_t seqs, int64_t tokens, int64_t max_tokens, int64_t group,
                         int64_t kv_heads, int64_t prefix, int64_t len, int64_t hd, int64_t* out) {
  const dnx::PagedSplit s =
      dnx::paged_split(seqs, tokens, max_tokens, group, kv_heads, prefix, len, false, (int)hd);
  const int64_t v[] = {s.prefix_items, s.own_items, s.prefix.runs, s.own.runs, s.prefix.blocks,
                       s.own.blocks, s.prefix.together, s.own.together, s.slots, s.splits(),
                       s.prefix.keys, s.own.keys, s.joined, dnx::kPagedItems};
  for (int i = 0; i < 14; i++) out[i] = v[i];
}
"""


@pytest.fixture(scope="module")
def split_of(tmp_path_factory):
    d = tmp_path_factory.mktemp("split")
    (d / "s.cpp").write_text(SOURCE)
    so = str(d / "s.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so, str(d / "s.cpp"),
                    "-I", os.path.join(ROOT, "dianoia_amd", "csrc")], check=True)
    f = ctypes.CDLL(so).split_of
    f.argtypes, f.restype = [ctypes.c_int64] * 8 + [ctypes.c_void_p], None

    def call(*args):
        out = (ctypes.c_int64 * 14)()
        f(*args, out)
        return list(out)
    return call


def places(items, blocks, kv, together):
    """(set, key head, block) of each workgroup, as paged_workgroup finds them."""
    for i in range(items):
        turn = i // 8
        unit, block = turn // blocks * 8 + i % 8, turn % blocks
        if together:
            yield unit // 8 // kv * 8 + unit % 8, unit // 8 % kv, block, i % 8
        else:
            yield unit // kv, unit % kv, block, i % 8


def test_every_block_has_a_workgroup(split_of):
    for seqs, each, group, kv, prefix, length, hd in itertools.product(
            (1, 3, 8, 64, 70), (1, 5, 70), (1, 4), (1, 2, 3, 8), (0, 65, 777, 8192), (0, 64, 500, 5000),
            (64, 128)):
        p_items, o_items, p_runs, o_runs, p_blocks, o_blocks, p_tog, o_tog, slots, splits, p_keys, o_keys, \
            joined, most = split_of(seqs, seqs * each, each, group, kv, prefix, length, hd)
        assert p_items % 8 == 0 and p_items + o_items <= most and splits <= 256
        assert not (hd == 128 and (p_tog or o_tog))
        parts = [(p_items, p_blocks, p_runs, p_tog)]
        if slots:            # blocks of all sequences in a row: one a unit
            parts.append((o_items, 1, slots * o_runs, o_tog) if o_tog else (0, 1, 0, 0))
        else:
            parts.append((o_items, o_blocks, seqs * o_runs, o_tog))
        for items, blocks, sets, together in parts:
            if items > 200000:
                continue
            seen = {}
            for s, h, b, xcd in places(items, blocks, kv, together):
                if s < sets:
                    assert (s, h, b) not in seen
                    seen[s, h, b] = xcd
            assert len(seen) == sets * kv * blocks
            if together:
                assert all(xcd == s % 8 for (s, _, _), xcd in seen.items())


def test_large_bounds_stay_within_a_launch(split_of):
    for kv, prefix, length, hd in itertools.product((1, 8, 32), (0, 300, 1 << 20), (1 << 14, 1 << 24), (64, 128)):
        for seqs in (4096, 1 << 17, (1 << 22) // kv):
            v = split_of(seqs, 8192, 4200, 2, kv, prefix, length, hd)
            assert 0 < v[0] + v[1] <= v[13]


def test_workspace_and_refusals_of_an_int8_cache():
    from dianoia_amd import _lib
    lib = _lib.load()
    a = 4096   # a pointer that no refused call reads

    def cache(**k):
        return ctypes.byref(_lib.PagedCacheStruct(**{**dict(
            keys=a, values=a, pages=64, page=16, kv_heads=2, hd=64, type=2, key_scales=a,
            value_scales=a), **k}))

    def batch(**k):
        return ctypes.byref(_lib.PagedBatchStruct(**{**dict(
            starts=a, lens=a, tables=a, prefix_pages=a, table_stride=4, prefix_len=1000, seqs=3, tokens=8,
            max_tokens=1, max_len=64), **k}))

    def run(c, b, q=a, out=a, ws=a, nbytes=1 << 30, heads=4, window=0):
        return lib.dnx_paged_attention(c, b, q, None, out, heads, window, ws, nbytes, None)

    need = lib.dnx_paged_attention_workspace_bytes(cache(), batch(), 4)
    assert need > 0 and need % (8 * 4 * (64 + 2) * 4) == 0
    for bad in (dict(key_scales=None), dict(value_scales=None), dict(key_scales=a + 4), dict(value_scales=a + 8),
                dict(type=3), dict(keys=a + 8), dict(hd=96), dict(page=8)):
        assert lib.dnx_paged_attention_workspace_bytes(cache(**bad), batch(), 4) == -1, bad
        assert run(cache(**bad), batch()) == -1, bad
    for bad in (dict(q=None), dict(out=None), dict(q=a + 4), dict(ws=None), dict(nbytes=need - 1), dict(heads=3),
                dict(window=-1)):
        assert run(cache(), batch(), **bad) == -1, bad
    assert run(cache(), batch(tokens=0)) == 0
