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
