"""A C caller's dnx_paged_cache without the scales' fields at its end, as float32 and
bf16 caches need it: the calls read nothing past it. The struct ends where memory
does, in a child process that sees no GPU, so that a call that passes its checks
ends at the launch."""

import os
import signal
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import ctypes, mmap, sys
from dianoia_amd import _lib
lib = _lib.load()
libc = ctypes.CDLL(None, use_errno=True)
size = mmap.PAGESIZE
memory = mmap.mmap(-1, 2 * size)
at = ctypes.addressof(ctypes.c_char.from_buffer(memory))
libc.mprotect.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
assert libc.mprotect(at + size, size, 0) == 0

class Short(ctypes.Structure):
    _fields_ = _lib.PagedCacheStruct._fields_[:7]

a = 4096   # a pointer that nothing reads
cache = at + size - ctypes.sizeof(Short)
Short.from_address(cache).__init__(keys=a, values=a, pages=64, page=16, kv_heads=2, hd=64,
                                   type=int(sys.argv[2]))
if sys.argv[1] == "append":
    rc = lib.dnx_paged_append(cache, None, 0, None, a, 128, a, 128, None, None, None, 0, None, a, 0, 2,
                              1e-6, None)
elif sys.argv[1] == "read":
    rc = lib.dnx_paged_read(cache, a, a, 128, a, 128, 2, None)
else:
    batch = _lib.PagedBatchStruct(a, a, a, None, 4, 0, 1, 1, 1, 64)
    need = lib.dnx_paged_attention_workspace_bytes(cache, ctypes.byref(batch), 4)
    assert need >= 0
    rc = lib.dnx_paged_attention(cache, ctypes.byref(batch), a, None, a, 4, 0, a, need + 64, None)
print("returned", rc)
"""


@pytest.mark.parametrize("kind", [0, 1])
@pytest.mark.parametrize("call", ["append", "read", "attention"])
def test_nothing_is_read_past_a_float_cache(call, kind):
    env = {**os.environ, "HIP_VISIBLE_DEVICES": "-1", "PYTHONPATH": ROOT}
    r = subprocess.run([sys.executable, "-c", CHILD, call, str(kind)], env=env, cwd=ROOT,
                       capture_output=True, text=True, timeout=300)
    assert r.returncode != -signal.SIGSEGV, (call, kind)
    assert r.returncode == 0 and r.stdout.startswith("returned"), r.stderr
    assert r.stdout.split()[1] != "-1", "refused by a check, not at the launch"
