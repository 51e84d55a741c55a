"""How the paged attention deals keys to workgroups (paged_split.h), compiled
for the CPU: every key in one run, runs of whole steps, no more partial results
than the second launch adds, and the workspace that a call asks for."""

import ctypes
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "paged_split.h"
extern "C" void split_of(int64_t seqs, int64_t tokens, int64_t max_tokens, int64_t group,
                         int64_t kv_heads, int64_t prefix, int64_t len, int64_t f32, int64_t* out) {
  const dnx::PagedSplit s =
      dnx::paged_split(seqs, tokens, max_tokens, group, kv_heads, prefix, len, f32 != 0);
  const int64_t v[] = {s.prefix.blocks, s.own.blocks, s.prefix.runs, s.prefix.keys, s.own.runs,
                       s.own.keys, s.splits(), s.joined};
  for (int i = 0; i < 8; i++) out[i] = v[i];
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
        out = (ctypes.c_int64 * 8)()
        f(*args, out)
        return list(out)
    return call


def test_every_key_has_a_run(split_of):
    for seqs, each, group, kv, prefix, length, f32 in itertools.product(
            (1, 3, 64, 300), (1, 5, 70), (1, 3, 8, 33), (1, 2, 8), (0, 1, 63, 65, 777, 8192, 200000),
            (0, 1, 64, 500, 2048, 100000), (0, 1)):
        tokens = seqs * each
        pr, orows, ps, prun, os_, orun, total, joined = split_of(seqs, tokens, each, group, kv, prefix,
                                                                length, f32)
        assert total == ps + os_ <= 256
        if joined:       # one run of both, in which the own keys begin at a step
            assert (ps, os_) == (0, 1) and joined % 64 == 0 and prefix <= joined < prefix + 64
            assert joined + length <= orun <= 384 and orows >= 1
            continue
        for keys, splits, run in ((prefix, ps, prun), (length, os_, orun)):
            assert run % 64 == 0 and run > 0
            if keys == 0:
                assert splits == 0
            else:
                assert (splits - 1) * run < keys <= splits * run
        assert orows >= 1 and pr >= 1


def test_workspace_and_refusals():
    """The sizes and refusals of the C entry points, none of which launches."""
    from dianoia_amd import _lib
    lib = _lib.load()
    a = 4096   # a pointer that no refused call reads

    def cache(**k):
        return _lib.PagedCacheStruct(**{**dict(keys=a, values=a, pages=64, page=16, kv_heads=2, hd=64,
                                               type=0), **k})

    def batch(**k):
        return _lib.PagedBatchStruct(**{**dict(starts=a, lens=a, tables=a, prefix_pages=a, table_stride=4,
                                               prefix_len=1000, seqs=3, tokens=8, max_tokens=1,
                                               max_len=64), **k})

    def size(c, b, heads=4):
        return lib.dnx_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), heads)

    def run(c, b, heads=4, q=a, gate=None, out=a, window=0, ws=a, nbytes=1 << 30):
        return lib.dnx_paged_attention(ctypes.byref(c), ctypes.byref(b), q, gate, out, heads, window,
                                       ws, nbytes, None)

    need = size(cache(), batch())
    assert need > 0 and need % (8 * 4 * (64 + 2) * 4) == 0
    assert size(cache(), batch(prefix_len=0)) == 0        # one run: no partial results
    bad_caches = [dict(keys=None), dict(values=None), dict(keys=a + 8), dict(pages=0), dict(page=8),
                  dict(page=24), dict(page=8192), dict(pages=1 << 30), dict(kv_heads=0), dict(kv_heads=1025),
                  dict(hd=32), dict(hd=96), dict(hd=256), dict(type=2), dict(type=-1)]
    bad_batches = [dict(starts=None), dict(lens=None), dict(tables=None), dict(prefix_pages=None),
                   dict(seqs=0), dict(tokens=-1), dict(max_tokens=0), dict(max_len=-1),
                   dict(prefix_len=-1), dict(prefix_len=1 << 40), dict(table_stride=-1),
                   dict(tokens=1 << 30)]
    for bad in bad_caches:
        assert size(cache(**bad), batch()) == -1 and run(cache(**bad), batch()) == -1, bad
    for bad in bad_batches:
        assert size(cache(), batch(**bad)) == -1 and run(cache(), batch(**bad)) == -1, bad
    for heads in (0, 3, -2, 1 << 20):
        assert size(cache(), batch(), heads) == -1 and run(cache(), batch(), heads=heads) == -1
    for bad in (dict(q=None), dict(out=None), dict(q=a + 4), dict(out=a + 8), dict(gate=a + 2),
                dict(window=-1), dict(window=1 << 31), dict(ws=None), dict(ws=a + 4), dict(nbytes=need - 1)):
        assert run(cache(), batch(), **bad) == -1, bad
    assert run(cache(), batch(tokens=0)) == 0
    assert lib.dnx_paged_attention(None, ctypes.byref(batch()), a, None, a, 4, 0, a, 1 << 30, None) == -1
    assert lib.dnx_paged_attention(ctypes.byref(cache()), None, a, None, a, 4, 0, a, 1 << 30, None) == -1

    def append(c=cache(), **k):
        v = {**dict(q=a, qs=256, qo=a, k=a, ks=128, v=a, vs=128, qn=a, kn=a, rope=a, rr=100, pos=a, slots=a,
                    heads=4, n=2, eps=1e-6, st=None), **k}
        return lib.dnx_paged_append(ctypes.byref(c), *v.values())

    for bad in bad_caches:
        assert append(cache(**bad)) == -1, bad
    for bad in (dict(qs=255), dict(qs=252), dict(qo=None), dict(qo=a + 4), dict(k=None), dict(k=a + 4), dict(ks=127),
                dict(ks=130), dict(v=None), dict(vs=64), dict(qn=a + 4), dict(kn=a + 8), dict(rope=a + 4),
                dict(rr=0), dict(pos=None), dict(slots=None), dict(slots=a + 1), dict(heads=0), dict(heads=-1),
                dict(n=-1), dict(n=1 << 30)):
        assert append(**bad) == -1, bad
    assert append(n=0) == 0


def test_limits_of_sizes():
    """Sizes whose products leave 32 or 64 bits, or a launch's threads, are
    refused; none of these calls launches."""
    from dianoia_amd import _lib
    lib = _lib.load()
    a = 4096

    def size(tokens=8, heads=4, pages=64, prefix=1000, length=64):
        c = _lib.PagedCacheStruct(keys=a, values=a, pages=pages, page=16, kv_heads=2, hd=64, type=0)
        b = _lib.PagedBatchStruct(starts=a, lens=a, tables=a, prefix_pages=a, table_stride=4,
                                  prefix_len=prefix, seqs=3, tokens=tokens, max_tokens=1, max_len=length)
        return lib.dnx_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), heads)

    assert size() > 0 and size(tokens=1 << 22, heads=14) > 0
    assert size(tokens=1 << 22, heads=16) == -1
    for pages in (1 << 27, 1 << 60, (1 << 60) + 1):
        assert size(pages=pages) == -1
    assert size(prefix=1 << 30, length=1 << 30) == -1
    for rows in (1 << 22, 1 << 40):
        assert lib.dnx_quantize_i8r(a, a, a, rows, 64, 64, None) == -1
        assert lib.dnx_gemm_i8r(a, a, a, a, a, rows, 64, 2, None) == -1
        assert lib.dnx_gemm_i8r(a, a, a, a, a, 8, 64, rows, None) == -1
    assert lib.dnx_gemm_i8r(a, a, a, a, a, (1 << 22) - 1, 64, (1 << 22) - 1, None) == -1


def test_python_refusals():
    import torch

    from dianoia_amd import device as D
    k = torch.zeros(4, 16, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        D.PagedCache(k, k.clone())
    for bad in (torch.zeros(4, 16, 128), torch.zeros(4, 8, 2, 64), torch.zeros(4, 24, 2, 64),
                torch.zeros(4, 16, 2, 32), torch.zeros(4, 16, 2, 64).half(), torch.zeros(0, 16, 2, 64)):
        with pytest.raises(ValueError):
            D.PagedCache(bad, bad.clone())
    with pytest.raises(ValueError):
        D.PagedCache(k, torch.zeros(4, 16, 2, 128))
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    for args in ((i(4).long(), i(3), i(3, 2), 3, 1, 5), (i(3), i(3), i(3, 2), 3, 1, 5),
                 (i(4), i(3), i(2, 2), 3, 1, 5), (i(4), i(3), i(6), 3, 1, 5), (i(4), i(3), i(3, 2), -1, 1, 5),
                 (i(4), i(3), i(3, 2), 3, 0, 5), (i(4), i(3), i(3, 2), 3, 1, 5)):
        with pytest.raises(ValueError):   # the last: not in HBM
            D.PagedBatch(*args)


FIT = """
#include "paged_split.h"
extern "C" void fit_of(int64_t seqs, int64_t tokens, int64_t max_tokens, int64_t group,
                       int64_t kv_heads, int64_t prefix, int64_t len, int64_t f32, int64_t* out) {
  const dnx::PagedSplit s =
      dnx::paged_split(seqs, tokens, max_tokens, group, kv_heads, prefix, len, f32 != 0);
  const int64_t v[] = {s.prefix_items, s.own_items, s.slots, s.prefix.runs, s.prefix.keys, s.own.runs,
                       s.own.keys, s.splits(), s.own.wide, s.own.blocks};
  for (int i = 0; i < 10; i++) out[i] = v[i];
}
extern "C" int place_of(const int32_t* starts, int b, int live, int group, int block) {
  return dnx::paged_slot(starts, b, live, group, block);
}
extern "C" int sequence_of(const int32_t* starts, int seqs, int live, int group, int block, int slot) {
  return dnx::paged_sequence(starts, seqs, live, group, block, slot);
}
"""


@pytest.fixture(scope="module")
def fit(tmp_path_factory):
    d = tmp_path_factory.mktemp("fit")
    (d / "f.cpp").write_text(FIT)
    so = str(d / "f.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", so, str(d / "f.cpp"),
                    "-I", os.path.join(ROOT, "dianoia_amd", "csrc")], check=True)
    lib = ctypes.CDLL(so)
    lib.fit_of.argtypes, lib.fit_of.restype = [ctypes.c_int64] * 8 + [ctypes.c_void_p], None
    lib.place_of.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 4
    lib.sequence_of.argtypes = [ctypes.c_void_p] + [ctypes.c_int] * 5
    return lib


def test_every_call_fits_a_launch(fit):
    """Whatever the bounds, up to 2^22 key heads of sequences and 2^26 rows: no
    more workgroups than a launch may have, every key in one run, at most 256
    runs, and where a launch holds a place for every block, that place."""
    limit = 0xffffffff // 256
    out = (ctypes.c_int64 * 10)()
    for seqs, kv, group, tokens, most, prefix, length, f32 in itertools.product(
            (1, 64, 4096, 1 << 20), (1, 8, 31, 1024), (1, 4, 64), (1, 2000, 16384, 1 << 22),
            (1, 20, 8192, 1 << 22), (0, 300, 1 << 25, 1 << 30), (0, 200, 131072, 1 << 30), (0, 1)):
        if tokens * kv * group >= 1 << 26 or seqs * kv > 1 << 22 or prefix + length >= 1 << 31:
            continue
        args = seqs, tokens, min(most, tokens), group, kv, prefix, length, f32
        fit.fit_of(*args, out)
        prefix_items, own_items, slots, pr, pk, orun, ok, total, wide, blocks = out
        assert 0 <= prefix_items + own_items <= limit, args
        assert total == pr + orun <= 256
        if pr:
            assert pk % 64 == 0 and (pr - 1) * pk < prefix <= pr * pk < 1 << 31, args
        if orun:
            begin = -(-prefix // 64) * 64 if prefix and not pr else 0
            assert ok % 64 == 0 and (orun - 1) * ok < begin + length <= orun * ok < 1 << 31, args
            if slots:
                assert slots >= tokens * group // (64 if wide else 16) + seqs
                assert own_items == slots * kv * orun
            else:
                assert own_items == -(-seqs * kv * orun // 8) * 8 * blocks


@pytest.mark.parametrize("group,block", [(1, 16), (3, 16), (4, 64), (7, 64), (64, 16)])
def test_every_block_has_a_place(fit, group, block):
    """Blocks of all sequences in a row: each finds its sequence, whatever the
    tokens of each are, and no place lies outside."""
    import random
    rng = random.Random(group * block)
    for seqs in (1, 2, 5, 100):
        for most in (0, 1, 17, 300):
            counts = [rng.choice([0, 0, 1, rng.randint(0, most)]) if most else 0 for _ in range(seqs)]
            starts = [0]
            for c in counts:
                starts.append(starts[-1] + c)
            live = starts[-1]
            a = (ctypes.c_int32 * len(starts))(*starts)
            places = live * group // block + seqs
            found = set()
            for slot in range(places):
                b = fit.sequence_of(a, seqs, live, group, block, slot)
                at = slot - fit.place_of(a, b, live, group, block)
                assert 0 <= b < seqs and at >= 0
                if at * block < counts[b] * group:
                    assert (b, at) not in found
                    found.add((b, at))
            assert found == {(b, i) for b, c in enumerate(counts)
                             for i in range(-(-c * group // block))}


def test_bounds_beyond_a_launch_are_refused_by_both():
    """More key heads of sequences than a launch has workgroups: no size is given
    for what the call would refuse."""
    from dianoia_amd import _lib
    lib = _lib.load()
    a = 4096
    c = _lib.PagedCacheStruct(keys=a, values=a, pages=64, page=16, kv_heads=32, hd=64, type=0)
    for seqs, ok in ((1 << 17, True), (1 << 20, False)):
        b = _lib.PagedBatchStruct(starts=a, lens=a, tables=a, prefix_pages=a, table_stride=4,
                                  prefix_len=1000, seqs=seqs, tokens=8, max_tokens=8, max_len=64)
        size = lib.dnx_paged_attention_workspace_bytes(ctypes.byref(c), ctypes.byref(b), 32)
        assert (size > 0) == ok
        if not ok:
            assert size == -1
            assert lib.dnx_paged_attention(ctypes.byref(c), ctypes.byref(b), a, None, a, 32, 0, a,
                                           1 << 40, None) == -1


def test_blocks_in_a_row_where_many_would_be_empty(fit):
    """A step of single tokens and a batch of equal prompts have a place for every
    block; one prompt among single tokens, and bounds above the batch, do not."""
    out = (ctypes.c_int64 * 10)()

    def slots(seqs, tokens, most, length=1000, kv=8, group=4):
        fit.fit_of(seqs, tokens, most, group, kv, 0, length, 0, out)
        return out[2]

    assert slots(64, 64, 1) == 0 and slots(1, 1, 1) == 0 and slots(16, 16 * 512, 512) == 0
    assert slots(64, 575, 512) == 575 * 4 // 64 + 64
    assert slots(64, 64, 64) == 64 * 4 // 64 + 64
    assert slots(2, 40, 39) == 0 and slots(64, 64, 64, length=0) == 0


def test_arrays_off_their_alignment_are_refused():
    """A scalar load drops the last bits of an address: it would read other numbers."""
    from dianoia_amd import _lib
    lib = _lib.load()
    a = 4096
    c = _lib.PagedCacheStruct(keys=a, values=a, pages=64, page=16, kv_heads=2, hd=64, type=0)
    good = dict(starts=a, lens=a, tables=a, prefix_pages=a, table_stride=4, prefix_len=1000, seqs=3,
                tokens=8, max_tokens=1, max_len=64)
    size = lambda **k: lib.dnx_paged_attention_workspace_bytes(
        ctypes.byref(c), ctypes.byref(_lib.PagedBatchStruct(**{**good, **k})), 4)
    assert size() > 0
    for name in ("starts", "lens", "tables", "prefix_pages"):
        for off in (1, 2, 3):
            assert size(**{name: a + off}) == -1, (name, off)
        assert size(**{name: a + 4}) > 0
