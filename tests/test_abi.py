"""The drop-in boundary on the CPU: the library builds, loads, and exports
every symbol include/*.h declares. No compute call (no GPU here)."""

import ctypes
import os
import subprocess

import pytest

from dianoia_amd import _lib
from dianoia_amd import device as D

# The reference's GPU entry points that Dart binds (lib/src/gpu.dart:36-312):
# the matmul path, everything GpuLinear and the GPU layer's lifecycle,
# profiling and tuning calls reach, and the decoder's other layer steps.
REFERENCE_BOUND = [
    "lab_gpu_init", "lab_gpu_max_buffer_length", "lab_gpu_max_shared_memory",
    "lab_gpu_recommended_working_set", "lab_gpu_thermal_state", "lab_gpu_physical_memory",
    "lab_gpu_device_name", "lab_gpu_buffer", "lab_gpu_readback_buffer", "lab_gpu_wrap",
    "lab_gpu_wrap_copies", "lab_gpu_contents", "lab_gpu_release", "lab_gpu_live_buffers",
    "lab_gpu_set_decode_rows", "lab_gpu_set_q8_group", "lab_gpu_set_q8_vector",
    "lab_gpu_register_q8_head", "lab_gpu_set_profiling", "lab_gpu_profile", "lab_gpu_last_ms",
    "lab_gpu_begin", "lab_gpu_commit", "lab_gpu_wait", "lab_gpu_enc_matmul_q8",
    "lab_gpu_enc_matmul_q4", "lab_gpu_enc_swiglu", "lab_gpu_enc_rms_norm",
    "lab_gpu_enc_head_norm_rope", "lab_gpu_enc_conv", "lab_gpu_enc_attention", "lab_gpu_enc_copy",
    "lab_gpu_enc_add", "lab_gpu_enc_steer",
]


def test_library_is_built():
    assert os.path.exists(_lib.LIB_PATH), "run python -m dianoia_amd.build"


def test_exports_every_declared_symbol():
    declared = _lib.declared_symbols()
    assert len(declared) >= 40
    out = subprocess.run(["nm", "-D", "--defined-only", _lib.LIB_PATH], capture_output=True,
                         text=True, check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if " T " in line}
    missing = [s for s in declared if s not in exported]
    assert not missing, missing
    assert set(declared) == set(_lib.SIGNATURES), "ctypes signatures out of sync with headers"


def test_reference_gpu_abi_covered():
    declared = set(_lib.declared_symbols())
    assert [s for s in REFERENCE_BOUND if s not in declared] == []


def test_loads_with_ctypes():
    lib = _lib.load()
    for name in _lib.SIGNATURES:
        assert isinstance(getattr(lib, name), ctypes._CFuncPtr)


def test_no_oracle_in_product():
    # The product library must not link the CPU oracle or the reference.
    out = subprocess.run(["ldd", _lib.LIB_PATH], capture_output=True, text=True).stdout
    assert "lab_oracle" not in out and "lab_native" not in out
    syms = subprocess.run(["nm", "-D", _lib.LIB_PATH], capture_output=True, text=True).stdout
    assert "orc_" not in syms


@pytest.mark.parametrize("size", [D.gemm_panel_bytes, D.f6_panel_bytes, D.q4_f6pack_bytes,
                                  D.q8_f6pack_bytes, D.i8_panel_bytes, D.q8_i8pack_bytes])
def test_sizes_refuse_floats_also_after_integers(size):
    """The C ABI takes integers: a float shape is an error whether or not the
    same number was asked for as an integer before."""
    assert size(64, 96) > 0
    with pytest.raises(ctypes.ArgumentError):
        size(64.0, 96)


def test_int8_cache_and_sampling_refusals():
    """What the entry points of the int8 paged cache and of the sampling refuse,
    none of which launches."""
    lib = _lib.load()
    a = 4096   # a pointer that no refused call reads

    def cache(**k):
        return ctypes.byref(_lib.PagedCacheStruct(**{**dict(
            keys=a, values=a, pages=64, page=16, kv_heads=2, hd=64, type=2, key_scales=a,
            value_scales=a), **k}))

    def read(c=None, **k):
        v = {**dict(slots=a, k=a, ks=128, v=a, vs=128, n=2, st=None), **k}
        return lib.dnx_paged_read(c or cache(), *v.values())

    bad_caches = [dict(keys=None), dict(key_scales=None), dict(value_scales=None), dict(key_scales=a + 4),
                  dict(value_scales=a + 8), dict(type=3), dict(hd=32), dict(page=24), dict(kv_heads=0)]
    for bad in bad_caches:
        assert read(cache(**bad)) == -1, bad
        assert lib.dnx_paged_append(cache(**bad), None, 0, None, a, 128, a, 128, None, None, None, 0, None,
                                    a, 0, 2, 1e-6, None) == -1, bad
    for bad in (dict(slots=None), dict(slots=a + 2), dict(k=None, v=None), dict(k=a + 4), dict(v=a + 8),
                dict(ks=127), dict(ks=130), dict(vs=64), dict(n=-1), dict(n=(1 << 22) + 1)):
        assert read(**bad) == -1, bad
    assert read(cache(kv_heads=1024, hd=128), ks=1 << 17, vs=1 << 17, n=(1 << 17) + 1) == -1
    assert read(n=0) == 0

    def sample(**k):
        v = {**dict(logits=a, stride=100, u=a, t=a, k=a, p=a, low=a, out=a, rows=3, vocab=100, ws=a,
                    nbytes=1 << 30, st=None), **k}
        return lib.dnx_sample(*v.values())

    size = lib.dnx_sample_workspace_bytes
    assert size(3, 100) >= 0 and size(0, 1) == 0 and size(1 << 16, 1 << 20) >= 0
    for rows, vocab in ((-1, 100), (3, 0), (3, -1), ((1 << 16) + 1, 100), (3, (1 << 20) + 1)):
        assert size(rows, vocab) == -1 and sample(rows=rows, vocab=vocab, stride=1 << 21) == -1
    for bad in (dict(logits=None), dict(u=None), dict(out=None), dict(logits=a + 2), dict(u=a + 1),
                dict(t=a + 2), dict(k=a + 1), dict(p=a + 3), dict(low=a + 1), dict(out=a + 2),
                dict(stride=99), dict(stride=-1), dict(stride=1 << 41), dict(nbytes=-1)):
        assert sample(**bad) == -1, bad
    assert sample(rows=0) == 0
