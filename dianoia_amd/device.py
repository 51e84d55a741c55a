"""The dnx_* device launchers for torch tensors already in HBM.

torch supplies device memory and the stream (plumbing); the computation is
the library's HIP kernels. Every function enqueues on the current torch
stream (or ``stream``) and raises on a non-zero return code, before which
nothing was launched.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _lib


# Sizes depend on a shape alone. typed: 64.0 is refused also where 64 is held.
_size = functools.lru_cache(maxsize=1024, typed=True)


# A small kernel runs for less time than its launch takes from Python, so the
# checks below are few calls (torch.cuda.current_stream() builds an object,
# numel() * element_size() is two): a one-token 3072 x 1024 product went from
# 8.4 to 5.6 us a call.

def _stream(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _ptr(t: torch.Tensor | None) -> int | None:
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("device launchers take CUDA (HIP) tensors")
    if not t.is_contiguous():
        raise ValueError("device launchers take contiguous tensors")
    return t.data_ptr()


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise RuntimeError(f"{what} failed with code {rc}")


def _need(what: str, **operands) -> None:
    """Refuses, before any launch, an operand tensor smaller than the bytes
    the kernel will touch for the given shape (the C ABI takes bare
    pointers and cannot tell)."""
    for name, (t, nbytes) in operands.items():
        if t is not None and t.nbytes < nbytes:
            raise ValueError(f"{what}: {name} holds {t.nbytes} bytes, the shape needs {nbytes}")


def quantize_q8(x: torch.Tensor, qs: torch.Tensor, scales: torch.Tensor, rows: int, cols: int,
                cols_pad: int, stream=None) -> None:
    _need("quantize_q8",
          x=(x, rows * cols * 4),
          qs=(qs, rows * cols_pad),
          scales=(scales, rows * (cols_pad // 32) * 4))
    _check(_lib.load().dnx_quantize_q8(_ptr(x), _ptr(qs), _ptr(scales), rows, cols, cols_pad,
                                       _stream(stream)), "dnx_quantize_q8")


def quantize_q8_bf16(w: torch.Tensor, qs: torch.Tensor, scales: torch.Tensor, rows: int,
                     cols: int, cols_pad: int, stream=None) -> None:
    _check(_lib.load().dnx_quantize_q8_bf16(_ptr(w), _ptr(qs), _ptr(scales), rows, cols,
                                            cols_pad, _stream(stream)), "dnx_quantize_q8_bf16")


def quantize_q4(w: torch.Tensor, qs: torch.Tensor, scales: torch.Tensor, rows: int, cols: int,
                stream=None) -> None:
    """lab_quantize_q4 on the GPU: fp32 [rows][cols] -> nibbles [rows][cols/2] + fp16 bits."""
    _check(_lib.load().dnx_quantize_q4(_ptr(w), _ptr(qs), _ptr(scales), rows, cols,
                                       _stream(stream)), "dnx_quantize_q4")


def q6k_to_q8(blocks: torch.Tensor, qs: torch.Tensor, scales: torch.Tensor, rows: int, cols: int,
              stream=None) -> None:
    """Q6_K super-blocks -> the engine's Q8 (dequantizeQ6K + lab_quantize_q8, fused)."""
    _check(_lib.load().dnx_q6k_to_q8(_ptr(blocks), _ptr(qs), _ptr(scales), rows, cols,
                                     _stream(stream)), "dnx_q6k_to_q8")


def split_q8_0(blocks: torch.Tensor, qs: torch.Tensor, scales: torch.Tensor, count: int,
               stream=None) -> None:
    """GGUF Q8_0 blocks -> int8 values + fp32 scales (splitQ8_0, gguf.dart:270-282)."""
    _check(_lib.load().dnx_split_q8_0(_ptr(blocks), _ptr(qs), _ptr(scales), count,
                                      _stream(stream)), "dnx_split_q8_0")


def split_q4_0(blocks: torch.Tensor, qs: torch.Tensor, scales: torch.Tensor, count: int,
               stream=None) -> None:
    """GGUF Q4_0 blocks -> nibble bytes + fp16 scale bits (splitQ4_0, gguf.dart:208-218)."""
    _check(_lib.load().dnx_split_q4_0(_ptr(blocks), _ptr(qs), _ptr(scales), count,
                                      _stream(stream)), "dnx_split_q4_0")


def quantize_q4_bf16(w: torch.Tensor, qs: torch.Tensor, scales: torch.Tensor, rows: int,
                     cols: int, stream=None) -> None:
    """BF16 bits widened (p << 16), then lab_quantize_q4, in one kernel."""
    _check(_lib.load().dnx_quantize_q4_bf16(_ptr(w), _ptr(qs), _ptr(scales), rows, cols,
                                            _stream(stream)), "dnx_quantize_q4_bf16")


def gemv_q8(qs, scales, x, y, rows: int, cols: int, n: int = 1, stream=None) -> None:
    _need("gemv_q8",
          qs=(qs, rows * cols),
          scales=(scales, rows * (cols // 32) * 4),
          x=(x, n * cols * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemv_q8(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                   _stream(stream)), "dnx_gemv_q8")


def gemv_q4(qs, scales, x, y, rows: int, cols: int, n: int = 1, stream=None) -> None:
    _need("gemv_q4",
          qs=(qs, rows * cols // 2),
          scales=(scales, rows * (cols // 32) * 2),
          x=(x, n * cols * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemv_q4(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                   _stream(stream)), "dnx_gemv_q4")


def gemv_q8_float(qs, scales, x, y, rows: int, cols: int, n: int = 1, stream=None) -> None:
    """Float-input GEMV (lab_gemm_q8 mode 0), any n."""
    _need("gemv_q8_float",
          qs=(qs, rows * cols),
          scales=(scales, rows * (cols // 32) * 4),
          x=(x, n * cols * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemv_q8_float(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                         _stream(stream)), "dnx_gemv_q8_float")


def gemv_q4_float(qs, scales, x, y, rows: int, cols: int, n: int = 1, stream=None) -> None:
    """Float-input GEMV (lab_gemm_q4 mode 0), any n."""
    _need("gemv_q4_float",
          qs=(qs, rows * cols // 2),
          scales=(scales, rows * (cols // 32) * 2),
          x=(x, n * cols * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemv_q4_float(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                         _stream(stream)), "dnx_gemv_q4_float")


def gemv_argmax_workspace(device="cuda") -> torch.Tensor:
    """Zeroed workspace for the fused argmax GEMV; completed calls leave it zero."""
    nbytes = int(_lib.load().dnx_gemv_argmax_workspace_bytes())
    return torch.zeros(nbytes, dtype=torch.uint8, device=device)


def gemv_q8_argmax(qs, scales, x, y, out, workspace, rows: int, cols: int, stream=None) -> None:
    _check(_lib.load().dnx_gemv_q8_argmax(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols,
                                          _ptr(out), _ptr(workspace), _stream(stream)),
           "dnx_gemv_q8_argmax")


def gemv_q4_argmax(qs, scales, x, y, out, workspace, rows: int, cols: int, stream=None) -> None:
    _check(_lib.load().dnx_gemv_q4_argmax(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols,
                                          _ptr(out), _ptr(workspace), _stream(stream)),
           "dnx_gemv_q4_argmax")


def gate_up_q8(gq, gs, uq, us, x, h, rows: int, cols: int, n: int = 1, u=None,
               stream=None) -> None:
    _check(_lib.load().dnx_gate_up_q8(_ptr(gq), _ptr(gs), _ptr(uq), _ptr(us), _ptr(x), _ptr(h),
                                      _ptr(u), rows, cols, n, _stream(stream)), "dnx_gate_up_q8")


def gate_up_q4(gq, gs, uq, us, x, h, rows: int, cols: int, n: int = 1, u=None,
               stream=None) -> None:
    _check(_lib.load().dnx_gate_up_q4(_ptr(gq), _ptr(gs), _ptr(uq), _ptr(us), _ptr(x), _ptr(h),
                                      _ptr(u), rows, cols, n, _stream(stream)), "dnx_gate_up_q4")


def gemv_q8h(qs, scales, x, y, rows: int, cols: int, n: int = 1, stream=None) -> None:
    """Q8 GEMV with fp16 block scales (uint16 bits, the GGUF Q8_0 d)."""
    _check(_lib.load().dnx_gemv_q8h(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                    _stream(stream)), "dnx_gemv_q8h")


def gemv_q8h_argmax(qs, scales, x, y, out, workspace, rows: int, cols: int, stream=None) -> None:
    _check(_lib.load().dnx_gemv_q8h_argmax(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols,
                                           _ptr(out), _ptr(workspace), _stream(stream)),
           "dnx_gemv_q8h_argmax")


def gate_up_q8h(gq, gs, uq, us, x, h, rows: int, cols: int, n: int = 1, u=None,
                stream=None) -> None:
    _check(_lib.load().dnx_gate_up_q8h(_ptr(gq), _ptr(gs), _ptr(uq), _ptr(us), _ptr(x), _ptr(h),
                                       _ptr(u), rows, cols, n, _stream(stream)), "dnx_gate_up_q8h")


def copy_regions(regions, stream=None) -> None:
    """Byte copies in one launch: regions is a list of (src_ptr, dst_ptr,
    bytes) with device or pinned-host pointers (ints)."""
    count = len(regions)
    P = ctypes.c_void_p * max(count, 1)
    src = P(*[r[0] for r in regions])
    dst = P(*[r[1] for r in regions])
    nb = (ctypes.c_int64 * max(count, 1))(*[int(r[2]) for r in regions])
    _check(_lib.load().dnx_copy_regions(ctypes.cast(src, ctypes.c_void_p), ctypes.cast(dst, ctypes.c_void_p),
                                        ctypes.cast(nb, ctypes.c_void_p), count, _stream(stream)),
           "dnx_copy_regions")


def gemv_multi(fmt: str, mats, x, ys, cols: int, stream=None) -> None:
    """Up to 4 one-token GEMVs over the same x in one launch: mats is a list of
    (qs, scales, rows), ys the matching outputs; fmt "q8", "q4" or "q8h"."""
    segs = len(mats)
    P = ctypes.c_void_p * max(segs, 1)
    qs = P(*[_ptr(m[0]) for m in mats])
    sc = P(*[_ptr(m[1]) for m in mats])
    yp = P(*[_ptr(y) for y in ys])
    rows = (ctypes.c_int64 * max(segs, 1))(*[int(m[2]) for m in mats])
    name = {"q8": "dnx_gemv_multi_q8", "q4": "dnx_gemv_multi_q4", "q8h": "dnx_gemv_multi_q8h"}[fmt]
    _check(getattr(_lib.load(), name)(ctypes.cast(qs, ctypes.c_void_p), ctypes.cast(sc, ctypes.c_void_p),
                                      ctypes.cast(yp, ctypes.c_void_p), ctypes.cast(rows, ctypes.c_void_p),
                                      segs, _ptr(x), cols, _stream(stream)), name)


def gemv_add(fmt: str, qs, scales, x, y, resid, rows: int, cols: int, stream=None) -> None:
    """One-token GEMV whose epilogue also adds y into resid (fmt "q8" or "q4")."""
    name = {"q8": "dnx_gemv_add_q8", "q4": "dnx_gemv_add_q4"}[fmt]
    _check(getattr(_lib.load(), name)(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), _ptr(resid), rows,
                                      cols, _stream(stream)), name)


def gate_up_norm(fmt: str, gq, gs, uq, us, x, norm_w, norm_out, eps: float, h, u, rows: int,
                 cols: int, stream=None) -> None:
    """The gate/up pair and glue on RMSNorm(x) * norm_w, which also goes to norm_out."""
    name = {"q8": "dnx_gate_up_norm_q8", "q4": "dnx_gate_up_norm_q4"}[fmt]
    _check(getattr(_lib.load(), name)(_ptr(gq), _ptr(gs), _ptr(uq), _ptr(us), _ptr(x), _ptr(norm_w),
                                      _ptr(norm_out), eps, _ptr(h), _ptr(u), rows, cols,
                                      _stream(stream)), name)


def gemv_multi_norm(fmt: str, mats, x, norm_w, norm_out, eps: float, ys, cols: int,
                    stream=None) -> None:
    """gemv_multi on RMSNorm(x) * norm_w, which also goes to norm_out."""
    segs = len(mats)
    P = ctypes.c_void_p * max(segs, 1)
    qs = P(*[_ptr(m[0]) for m in mats])
    sc = P(*[_ptr(m[1]) for m in mats])
    yp = P(*[_ptr(y) for y in ys])
    rows = (ctypes.c_int64 * max(segs, 1))(*[int(m[2]) for m in mats])
    name = {"q8": "dnx_gemv_multi_norm_q8", "q4": "dnx_gemv_multi_norm_q4"}[fmt]
    _check(getattr(_lib.load(), name)(ctypes.cast(qs, ctypes.c_void_p), ctypes.cast(sc, ctypes.c_void_p),
                                      ctypes.cast(yp, ctypes.c_void_p), ctypes.cast(rows, ctypes.c_void_p),
                                      segs, _ptr(x), _ptr(norm_w), _ptr(norm_out), eps, cols,
                                      _stream(stream)), name)


def gemm_q8_float(qs, scales, x, y, rows: int, cols: int, n: int, stream=None) -> None:
    """Float-input (mode 0) GEMM on bf16 MFMA, within fp32 rounding of the CPU."""
    _need("gemm_q8_float",
          qs=(qs, rows * cols),
          scales=(scales, rows * (cols // 32) * 4),
          x=(x, n * cols * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q8_float(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                         _stream(stream)), "dnx_gemm_q8_float")


def gemm_q4_float(qs, scales, x, y, rows: int, cols: int, n: int, stream=None) -> None:
    _need("gemm_q4_float",
          qs=(qs, rows * cols // 2),
          scales=(scales, rows * (cols // 32) * 2),
          x=(x, n * cols * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q4_float(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                         _stream(stream)), "dnx_gemm_q4_float")


def gemm_q8(qs, scales, xq, xsc, y, rows: int, cols: int, n: int, stream=None) -> None:
    _need("gemm_q8",
          qs=(qs, rows * cols),
          scales=(scales, rows * (cols // 32) * 4),
          xq=(xq, n * cols),
          xsc=(xsc, n * (cols // 32) * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q8(_ptr(qs), _ptr(scales), _ptr(xq), _ptr(xsc), _ptr(y), rows,
                                   cols, n, _stream(stream)), "dnx_gemm_q8")


def gemm_q4(qs, scales, xq, xsc, y, rows: int, cols: int, n: int, stream=None) -> None:
    _need("gemm_q4",
          qs=(qs, rows * cols // 2),
          scales=(scales, rows * (cols // 32) * 2),
          xq=(xq, n * cols),
          xsc=(xsc, n * (cols // 32) * 4),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q4(_ptr(qs), _ptr(scales), _ptr(xq), _ptr(xsc), _ptr(y), rows,
                                   cols, n, _stream(stream)), "dnx_gemm_q4")


@_size
def gemm_panel_bytes(n: int, cols: int) -> int:
    return int(_lib.load().dnx_gemm_panel_bytes(n, cols))


def pack_panel(xq, xsc, panel, n: int, cols: int, stream=None) -> None:
    """xq int8 [n][cols] + xsc fp32 [n][cols/32] -> the GEMM's activation panel."""
    _check(_lib.load().dnx_pack_panel(_ptr(xq), _ptr(xsc), _ptr(panel), n, cols,
                                      _stream(stream)), "dnx_pack_panel")


def quantize_q8_panel(x, panel, n: int, cols: int, stream=None) -> None:
    """fp32 x [n][cols] quantized (lab_quantize_q8) straight into the GEMM's panel."""
    _need("quantize_q8_panel", x=(x, n * cols * 4), panel=(panel, gemm_panel_bytes(n, cols)))
    _check(_lib.load().dnx_quantize_q8_panel(_ptr(x), _ptr(panel), n, cols, _stream(stream)),
           "dnx_quantize_q8_panel")


def gemm_q8_panel(qs, scales, panel, y, rows: int, cols: int, n: int, stream=None) -> None:
    _check(_lib.load().dnx_gemm_q8_panel(_ptr(qs), _ptr(scales), _ptr(panel), _ptr(y), rows,
                                         cols, n, _stream(stream)), "dnx_gemm_q8_panel")


def gemm_q4_panel(qs, scales, panel, y, rows: int, cols: int, n: int, stream=None) -> None:
    _check(_lib.load().dnx_gemm_q4_panel(_ptr(qs), _ptr(scales), _ptr(panel), _ptr(y), rows,
                                         cols, n, _stream(stream)), "dnx_gemm_q4_panel")


@_size
def f6_panel_bytes(n: int, cols: int) -> int:
    return int(_lib.load().dnx_f6_panel_bytes(n, cols))


def quantize_q8_f6panel(x, panel, n: int, cols: int, stream=None) -> None:
    """fp32 x [n][cols] quantized (lab_quantize_q8) into the fp6 GEMM's panel."""
    _need("quantize_q8_f6panel", x=(x, n * cols * 4), panel=(panel, f6_panel_bytes(n, cols)))
    _check(_lib.load().dnx_quantize_q8_f6panel(_ptr(x), _ptr(panel), n, cols, _stream(stream)),
           "dnx_quantize_q8_f6panel")


def pack_f6panel(xq, xsc, panel, n: int, cols: int, stream=None) -> None:
    """xq int8 [n][cols] + xsc fp32 [n][cols/32] -> the fp6 GEMM's panel."""
    _need("pack_f6panel",
          xq=(xq, n * cols),
          xsc=(xsc, n * (cols // 32) * 4),
          panel=(panel, f6_panel_bytes(n, cols)))
    _check(_lib.load().dnx_pack_f6panel(_ptr(xq), _ptr(xsc), _ptr(panel), n, cols,
                                        _stream(stream)), "dnx_pack_f6panel")


def gemm_q4_f6(qs, scales, panel, y, rows: int, cols: int, n: int, stream=None) -> None:
    _need("gemm_q4_f6",
          qs=(qs, rows * cols // 2),
          scales=(scales, rows * (cols // 32) * 2),
          panel=(panel, f6_panel_bytes(n, cols)),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q4_f6(_ptr(qs), _ptr(scales), _ptr(panel), _ptr(y), rows, cols,
                                      n, _stream(stream)), "dnx_gemm_q4_f6")


@_size
def q4_f6pack_bytes(rows: int, cols: int) -> int:
    return int(_lib.load().dnx_q4_f6pack_bytes(rows, cols))


def pack_q4_f6(qs, scales, packed, rows: int, cols: int, stream=None) -> None:
    """Load-time re-encoding of Q4 weights for the fp6 GEMM (dnx_gemm_q4_f6p)."""
    _need("pack_q4_f6",
          qs=(qs, rows * cols // 2),
          scales=(scales, rows * (cols // 32) * 2),
          packed=(packed, q4_f6pack_bytes(rows, cols)))
    _check(_lib.load().dnx_pack_q4_f6(_ptr(qs), _ptr(scales), _ptr(packed), rows, cols,
                                      _stream(stream)), "dnx_pack_q4_f6")


def gemm_q4_f6p(packed, panel, y, rows: int, cols: int, n: int, stream=None) -> None:
    _need("gemm_q4_f6p",
          packed=(packed, q4_f6pack_bytes(rows, cols)),
          panel=(panel, f6_panel_bytes(n, cols)),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q4_f6p(_ptr(packed), _ptr(panel), _ptr(y), rows, cols, n,
                                       _stream(stream)), "dnx_gemm_q4_f6p")


def gemm_q4_f6s_multi(packs, ys, rows, panel, cols: int, n: int, stream=None) -> None:
    """The chunk GEMM over 1..4 prepacked matrices reading one panel, in one
    launch (each output bit-identical to its own gemm_q4_f6s)."""
    k = len(packs)
    if not (len(ys) == k == len(rows)):
        raise ValueError("gemm_q4_f6s_multi: one output and one row count per matrix")
    _need("gemm_q4_f6s_multi", panel=(panel, f6_panel_bytes(n, cols)))
    for j in range(k):
        _need("gemm_q4_f6s_multi", packed=(packs[j], q4_f6pack_bytes(rows[j], cols)),
              y=(ys[j], n * rows[j] * 4))
    pp = (ctypes.c_void_p * k)(*[_ptr(t) for t in packs])
    yp = (ctypes.c_void_p * k)(*[_ptr(t) for t in ys])
    rp = (ctypes.c_int64 * k)(*rows)
    _check(_lib.load().dnx_gemm_q4_f6s_multi(pp, yp, rp, k, _ptr(panel), cols, n,
                                             _stream(stream)), "dnx_gemm_q4_f6s_multi")


def gemm_q4_f6s(packed, panel, y, rows: int, cols: int, n: int, stream=None) -> None:
    """The prefill chunk GEMM (5..512 tokens) on prepacked Q4 weights."""
    _need("gemm_q4_f6s",
          packed=(packed, q4_f6pack_bytes(rows, cols)),
          panel=(panel, f6_panel_bytes(n, cols)),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q4_f6s(_ptr(packed), _ptr(panel), _ptr(y), rows, cols, n,
                                       _stream(stream)), "dnx_gemm_q4_f6s")


@_size
def q8_f6pack_bytes(rows: int, cols: int) -> int:
    return int(_lib.load().dnx_q8_f6pack_bytes(rows, cols))


def pack_q8_f6(qs, scales, packed, rows: int, cols: int, stream=None) -> None:
    """Load-time re-encoding of Q8 weights for the fp6 GEMM (dnx_gemm_q8_f6p)."""
    _need("pack_q8_f6",
          qs=(qs, rows * cols),
          scales=(scales, rows * (cols // 32) * 4),
          packed=(packed, q8_f6pack_bytes(rows, cols)))
    _check(_lib.load().dnx_pack_q8_f6(_ptr(qs), _ptr(scales), _ptr(packed), rows, cols,
                                      _stream(stream)), "dnx_pack_q8_f6")


def gemm_q8_f6p(packed, panel, y, rows: int, cols: int, n: int, stream=None) -> None:
    _need("gemm_q8_f6p",
          packed=(packed, q8_f6pack_bytes(rows, cols)),
          panel=(panel, f6_panel_bytes(n, cols)),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q8_f6p(_ptr(packed), _ptr(panel), _ptr(y), rows, cols, n,
                                       _stream(stream)), "dnx_gemm_q8_f6p")


@_size
def i8_panel_bytes(n: int, cols: int) -> int:
    return int(_lib.load().dnx_i8_panel_bytes(n, cols))


def quantize_q8_i8panel(x, panel, n: int, cols: int, stream=None) -> None:
    """fp32 x -> the int8 GEMM's activation panel (lab_quantize_q8's bits)."""
    _need("quantize_q8_i8panel", x=(x, n * cols * 4), panel=(panel, i8_panel_bytes(n, cols)))
    _check(_lib.load().dnx_quantize_q8_i8panel(_ptr(x), _ptr(panel), n, cols, _stream(stream)),
           "dnx_quantize_q8_i8panel")


@_size
def q8_i8pack_bytes(rows: int, cols: int) -> int:
    return int(_lib.load().dnx_q8_i8pack_bytes(rows, cols))


def pack_q8_i8(qs, scales, packed, rows: int, cols: int, stream=None) -> None:
    """Load-time re-encoding of Q8 weights for the int8 GEMM (dnx_gemm_q8_i8p)."""
    _need("pack_q8_i8",
          qs=(qs, rows * cols),
          scales=(scales, rows * (cols // 32) * 4),
          packed=(packed, q8_i8pack_bytes(rows, cols)))
    _check(_lib.load().dnx_pack_q8_i8(_ptr(qs), _ptr(scales), _ptr(packed), rows, cols,
                                      _stream(stream)), "dnx_pack_q8_i8")


def gemm_q8_i8p(packed, panel, y, rows: int, cols: int, n: int, stream=None) -> None:
    _need("gemm_q8_i8p",
          packed=(packed, q8_i8pack_bytes(rows, cols)),
          panel=(panel, i8_panel_bytes(n, cols)),
          y=(y, n * rows * 4))
    _check(_lib.load().dnx_gemm_q8_i8p(_ptr(packed), _ptr(panel), _ptr(y), rows, cols, n,
                                       _stream(stream)), "dnx_gemm_q8_i8p")


def gemm_q8_i8p_tile(rows: int, cols: int, n: int):
    """(weight rows, tokens) of the workgroup tile dnx_gemm_q8_i8p takes for
    a shape, or None for a shape it refuses."""
    r, t = ctypes.c_int(0), ctypes.c_int(0)
    rc = _lib.load().dnx_gemm_q8_i8p_tile(rows, cols, n, ctypes.byref(r), ctypes.byref(t))
    return None if rc != 0 else (r.value, t.value)


def argmax_workspace(n: int, device="cuda") -> torch.Tensor:
    nbytes = int(_lib.load().dnx_argmax_workspace_bytes(n))
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def argmax(v: torch.Tensor, out: torch.Tensor, workspace: torch.Tensor, stream=None) -> None:
    _check(_lib.load().dnx_argmax(_ptr(v), v.numel(), _ptr(out), _ptr(workspace),
                                  _stream(stream)), "dnx_argmax")


def swiglu(g: torch.Tensor, u: torch.Tensor, stream=None) -> None:
    _check(_lib.load().dnx_swiglu(_ptr(g), _ptr(u), g.numel(), _stream(stream)), "dnx_swiglu")


def swiglu_f6panel(g, u, panel, rows: int, cols: int, stream=None) -> None:
    """swiglu in place, and the fp6 panel of the result."""
    _need("swiglu_f6panel", g=(g, rows * cols * 4), u=(u, rows * cols * 4),
          panel=(panel, f6_panel_bytes(rows, cols)))
    _check(_lib.load().dnx_swiglu_f6panel(_ptr(g), _ptr(u), _ptr(panel), rows, cols,
                                          _stream(stream)), "dnx_swiglu_f6panel")


def rms_norm_f6panel(x, w, out, panel, rows: int, cols: int, eps: float, stream=None) -> None:
    """rms_norm (no accumulate), and the fp6 panel of its output."""
    _need("rms_norm_f6panel", x=(x, rows * cols * 4), w=(w, cols * 4),
          out=(out, rows * cols * 4), panel=(panel, f6_panel_bytes(rows, cols)))
    _check(_lib.load().dnx_rms_norm_f6panel(_ptr(x), _ptr(w), _ptr(out), _ptr(panel), rows, cols,
                                            eps, _stream(stream)), "dnx_rms_norm_f6panel")


def add_rms_norm_f6panel(m, x, w, out, panel, rows: int, cols: int, eps: float,
                         stream=None) -> None:
    """add_rms_norm, and the fp6 panel of its output."""
    _need("add_rms_norm_f6panel", m=(m, rows * cols * 4), x=(x, rows * cols * 4),
          w=(w, cols * 4), out=(out, rows * cols * 4), panel=(panel, f6_panel_bytes(rows, cols)))
    _check(_lib.load().dnx_add_rms_norm_f6panel(_ptr(m), _ptr(x), _ptr(w), _ptr(out),
                                                _ptr(panel), rows, cols, eps, _stream(stream)),
           "dnx_add_rms_norm_f6panel")


def gelu(x: torch.Tensor, stream=None) -> None:
    _check(_lib.load().dnx_gelu(_ptr(x), x.numel(), _stream(stream)), "dnx_gelu")


# ---- the decoder's other layer steps (lab_gpu_enc_* semantics, fp32)

def rms_norm(x, w, out, rows: int, cols: int, eps: float, accumulate: bool = False,
             stream=None) -> None:
    _check(_lib.load().dnx_rms_norm(_ptr(x), _ptr(w), _ptr(out), rows, cols, eps,
                                    1 if accumulate else 0, _stream(stream)), "dnx_rms_norm")


def head_norm_rope(x, x_stride: int, w, rope, rope_stride: int, heads: int, hd: int, n: int,
                   eps: float, stream=None) -> None:
    _check(_lib.load().dnx_head_norm_rope(_ptr(x), x_stride, _ptr(w), _ptr(rope), rope_stride,
                                          heads, hd, n, eps, _stream(stream)),
           "dnx_head_norm_rope")


def head_norm_rope2(x0, x0_stride: int, w0, heads0: int, x1, x1_stride: int, w1, heads1: int,
                    rope, rope_stride: int, hd: int, n: int, eps: float, stream=None) -> None:
    _check(_lib.load().dnx_head_norm_rope2(_ptr(x0), x0_stride, _ptr(w0), heads0, _ptr(x1),
                                           x1_stride, _ptr(w1), heads1, _ptr(rope), rope_stride,
                                           hd, n, eps, _stream(stream)), "dnx_head_norm_rope2")


def add_rms_norm(m, x, w, out, rows: int, cols: int, eps: float, stream=None) -> None:
    _check(_lib.load().dnx_add_rms_norm(_ptr(m), _ptr(x), _ptr(w), _ptr(out), rows, cols, eps,
                                        _stream(stream)), "dnx_add_rms_norm")


def short_conv(bcx, weight, history, y, width: int, k: int, n: int, stream=None) -> None:
    _check(_lib.load().dnx_short_conv(_ptr(bcx), _ptr(weight), _ptr(history), _ptr(y), width, k,
                                      n, _stream(stream)), "dnx_short_conv")


def attention(q, keys, values, gate, out, position: int, n: int, heads: int, kv_heads: int,
              hd: int, window: int = 0, stream=None) -> None:
    _check(_lib.load().dnx_attention(_ptr(q), _ptr(keys), _ptr(values),
                                     None if gate is None else _ptr(gate), _ptr(out), position, n,
                                     heads, kv_heads, hd, window, _stream(stream)),
           "dnx_attention")


def attention_f6panel(q, keys, values, gate, out, panel, position: int, n: int, heads: int,
                      kv_heads: int, hd: int, window: int = 0, stream=None) -> int:
    """attention, and the fp6 panel of out; returns the status (DNX_EINVAL
    where the call does not take the split path whose combine writes it)."""
    _need("attention_f6panel", panel=(panel, f6_panel_bytes(n, heads * hd)))
    return int(_lib.load().dnx_attention_f6panel(
        _ptr(q), _ptr(keys), _ptr(values), None if gate is None else _ptr(gate), _ptr(out),
        _ptr(panel), position, n, heads, kv_heads, hd, window, _stream(stream)))


def attention_rope(q, keys, values, gate, out, position: int, heads: int, kv_heads: int, hd: int,
                   window: int, q_norm, k_norm, rope_row, eps: float, stream=None) -> None:
    """One decode token: head norm + RoPE of q and of keys[position], folded
    into the split-key attention (q and the key row are normed in place)."""
    _check(_lib.load().dnx_attention_rope(_ptr(q), _ptr(keys), _ptr(values),
                                          None if gate is None else _ptr(gate), _ptr(out),
                                          position, heads, kv_heads, hd, window, _ptr(q_norm),
                                          _ptr(k_norm), _ptr(rope_row), eps, _stream(stream)),
           "dnx_attention_rope")


def add(src, dst, count: int, stream=None) -> None:
    _check(_lib.load().dnx_add(_ptr(src), _ptr(dst), count, _stream(stream)), "dnx_add")


def copy(src, dst, count: int, stream=None) -> None:
    _check(_lib.load().dnx_copy(_ptr(src), _ptr(dst), count, _stream(stream)), "dnx_copy")


def steer(x, v, rows: int, cols: int, mode: int, scale: float, stream=None) -> None:
    _check(_lib.load().dnx_steer(_ptr(x), _ptr(v), rows, cols, mode, scale, _stream(stream)),
           "dnx_steer")


def matmul_workspace(cols: int, n: int, device="cuda") -> torch.Tensor:
    """Device workspace for dnx_matmul_q8 / _q4 at this shape."""
    nbytes = int(_lib.load().dnx_matmul_workspace_bytes(cols, n))
    if nbytes < 0:
        raise RuntimeError(f"dnx_matmul_workspace_bytes({cols}, {n}) refused the shape")
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


def matmul_q8(qs, scales, x, y, rows: int, cols: int, n: int, int8_inputs: bool, workspace,
              stream=None) -> None:
    """The product route of lab_gpu_enc_matmul_q8 (dnx_matmul_q8)."""
    _check(_lib.load().dnx_matmul_q8(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                     int(int8_inputs), _ptr(workspace), workspace.numel(),
                                     _stream(stream)), "dnx_matmul_q8")


def matmul_q4(qs, scales, x, y, rows: int, cols: int, n: int, int8_inputs: bool, workspace,
              stream=None) -> None:
    """The product route of lab_gpu_enc_matmul_q4 (dnx_matmul_q4)."""
    _check(_lib.load().dnx_matmul_q4(_ptr(qs), _ptr(scales), _ptr(x), _ptr(y), rows, cols, n,
                                     int(int8_inputs), _ptr(workspace), workspace.numel(),
                                     _stream(stream)), "dnx_matmul_q4")


# ---- a batch of sequences at once: int8 rows and products, paged keys and values
#
# These run for a few microseconds, less than a careless launch takes from
# Python: sizes are compared in place, and an operand is named only once one
# is too small.

_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _device_of(t: torch.Tensor) -> int:
    """The current device, which has to be the tensor's."""
    d = t.get_device()
    if d < 0:
        raise ValueError("device launchers take CUDA (HIP) tensors")
    if d != torch._C._cuda_getDevice():
        raise ValueError(f"the tensor is on device {d}, not on the current one")
    return d


def _at(t: torch.Tensor | None, device: int) -> int | None:
    """The pointer of a contiguous tensor on that device."""
    if t is None:
        return None
    if t.get_device() != device:
        raise ValueError("device launchers take tensors of one CUDA (HIP) device")
    if not t.is_contiguous():
        raise ValueError("device launchers take contiguous tensors")
    return t.data_ptr()


def _on(device: int, stream) -> int:
    return torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream


def _refuse(*tensors) -> None:
    """Names what is wrong with one of them, which a caller has seen."""
    d = _device_of(tensors[0])
    for t in tensors:
        _at(t, d)
    raise ValueError("device launchers take tensors of one CUDA (HIP) device")


_F32, _I8, _I32 = torch.float32, torch.int8, torch.int32
_BF16 = (torch.bfloat16, torch.uint16, torch.int16)    # values, or their bits


def _types(name: str, **operands) -> None:
    """Names the operand that is not of its type, which a caller has seen."""
    for what, (t, kinds) in operands.items():
        kinds = kinds if isinstance(kinds, tuple) else (kinds,)
        if t is not None and t.dtype not in kinds:
            raise ValueError(f"{name}: {what} is {t.dtype}, not {' or '.join(map(str, kinds))}")


def _quantize_i8r(name: str, size: int, kinds, x, qs, scales, rows, cols, cols_pad, stream) -> None:
    if x.dtype not in kinds or qs.dtype is not _I8 or scales.dtype is not _F32:
        _types(name, x=(x, kinds), qs=(qs, _I8), scales=(scales, _F32))
    if x.nbytes < rows * cols * size or qs.nbytes < rows * cols_pad or scales.nbytes < rows * 4:
        _need(name, x=(x, rows * cols * size), qs=(qs, rows * cols_pad), scales=(scales, rows * 4))
    d = x.get_device()
    if (d < 0 or d != _current_device() or qs.get_device() != d or scales.get_device() != d
            or not (x.is_contiguous() and qs.is_contiguous() and scales.is_contiguous())):
        _refuse(x, qs, scales)
    rc = getattr(_lib._lib or _lib.load(), name)(
        x.data_ptr(), qs.data_ptr(), scales.data_ptr(), rows, cols, cols_pad,
        _raw_stream(d) if stream is None else stream.cuda_stream)
    if rc:
        _check(rc, name)


def quantize_i8r(x, qs, scales, rows: int, cols: int, cols_pad: int, stream=None) -> None:
    """fp32 rows -> int8 [rows][cols_pad] with one scale a row (value = code * scale)."""
    _quantize_i8r("dnx_quantize_i8r", 4, (_F32,), x, qs, scales, rows, cols, cols_pad, stream)


def quantize_i8r_bf16(x, qs, scales, rows: int, cols: int, cols_pad: int, stream=None) -> None:
    """bf16 rows (weights as they lie in a file: bfloat16, or its bits as 16-bit
    integers) -> int8 with one scale a row."""
    _quantize_i8r("dnx_quantize_i8r_bf16", 2, _BF16, x, qs, scales, rows, cols, cols_pad, stream)


def rms_norm_i8r(x, w, qs, scales, rows: int, cols: int, cols_pad: int, eps: float, m=None,
                 x_out=None, stream=None) -> None:
    """RMSNorm(s) * w as int8 with one scale a row; s = x, or x + m, which goes
    to x_out (x itself, m or another tensor)."""
    if (x.dtype is not _F32 or w.dtype is not _F32 or qs.dtype is not _I8
            or scales.dtype is not _F32 or (m is not None and m.dtype is not _F32)
            or (x_out is not None and x_out.dtype is not _F32)):
        _types("rms_norm_i8r", x=(x, _F32), w=(w, _F32), qs=(qs, _I8), scales=(scales, _F32),
               m=(m, _F32), x_out=(x_out, _F32))
    size = rows * cols * 4
    if (x.nbytes < size or w.nbytes < cols * 4 or qs.nbytes < rows * cols_pad
            or scales.nbytes < rows * 4 or (m is not None and m.nbytes < size)
            or (x_out is not None and x_out.nbytes < size)):
        _need("rms_norm_i8r", x=(x, size), w=(w, cols * 4), qs=(qs, rows * cols_pad),
              scales=(scales, rows * 4), m=(m, size), x_out=(x_out, size))
    d = x.get_device()
    if (d < 0 or d != _current_device() or w.get_device() != d or qs.get_device() != d
            or scales.get_device() != d or not (x.is_contiguous() and w.is_contiguous()
                                                and qs.is_contiguous() and scales.is_contiguous())):
        _refuse(x, w, qs, scales)
    rc = (_lib._lib or _lib.load()).dnx_rms_norm_i8r(
        x.data_ptr(), None if m is None else _at(m, d), None if x_out is None else _at(x_out, d),
        w.data_ptr(), qs.data_ptr(), scales.data_ptr(), rows, cols, cols_pad, eps,
        _raw_stream(d) if stream is None else stream.cuda_stream)
    if rc:
        _check(rc, "dnx_rms_norm_i8r")


def gemm_i8r(w, w_scale, x, x_scale, y, rows: int, cols: int, n: int, stream=None) -> None:
    """y [n][rows] = the int8 rows x times the int8 rows w, each with its scale."""
    if (w.dtype is not _I8 or x.dtype is not _I8 or w_scale.dtype is not _F32
            or x_scale.dtype is not _F32 or y.dtype is not _F32):
        _types("gemm_i8r", w=(w, _I8), w_scale=(w_scale, _F32), x=(x, _I8), x_scale=(x_scale, _F32),
               y=(y, _F32))
    if (w.nbytes < rows * cols or w_scale.nbytes < rows * 4 or x.nbytes < n * cols
            or x_scale.nbytes < n * 4 or y.nbytes < n * rows * 4):
        _need("gemm_i8r", w=(w, rows * cols), w_scale=(w_scale, rows * 4), x=(x, n * cols),
              x_scale=(x_scale, n * 4), y=(y, n * rows * 4))
    d = w.get_device()
    if (d < 0 or d != _current_device() or w_scale.get_device() != d or x.get_device() != d
            or x_scale.get_device() != d or y.get_device() != d
            or not (w.is_contiguous() and w_scale.is_contiguous() and x.is_contiguous()
                    and x_scale.is_contiguous() and y.is_contiguous())):
        _refuse(w, w_scale, x, x_scale, y)
    rc = (_lib._lib or _lib.load()).dnx_gemm_i8r(
        w.data_ptr(), w_scale.data_ptr(), x.data_ptr(), x_scale.data_ptr(), y.data_ptr(), rows, cols,
        n, _raw_stream(d) if stream is None else stream.cuda_stream)
    if rc:
        _check(rc, "dnx_gemm_i8r")


_CACHE_TYPES = {torch.float32: 0, torch.bfloat16: 1}   # DNX_F32, DNX_BF16


class PagedCache:
    """Keys and values in pages: two tensors [pages][page][kv_heads][hd],
    float32 or bfloat16 (dnx_paged_cache). Keeps the tensors, not copies."""

    def __init__(self, keys: torch.Tensor, values: torch.Tensor):
        if keys.dim() != 4 or keys.shape != values.shape or keys.dtype != values.dtype:
            raise ValueError("PagedCache: two tensors [pages][page][kv_heads][hd] of one type")
        if keys.dtype not in _CACHE_TYPES:
            raise ValueError("PagedCache: float32 or bfloat16")
        pages, page, kv_heads, hd = keys.shape
        if page < 16 or page > 4096 or page & (page - 1):
            raise ValueError("PagedCache: the page is a power of two from 16 to 4096")
        if hd not in (64, 128) or not 0 < kv_heads <= 1024 or not 0 < pages * page <= 0x7fffffff:
            raise ValueError("PagedCache: hd 64 or 128, up to 1024 heads, below 2^31 places")
        self.keys, self.values = keys, values
        self.page, self.kv_heads, self.hd = page, kv_heads, hd
        self.device = keys.get_device()
        self.struct = _lib.PagedCacheStruct(_ptr(keys), _at(values, self.device), pages, page,
                                            kv_heads, hd, _CACHE_TYPES[keys.dtype])
        self.ref = ctypes.addressof(self.struct)

    def check_device(self) -> int:
        if self.device != torch._C._cuda_getDevice():
            raise ValueError(f"the cache is on device {self.device}, not on the current one")
        return self.device


def _numbers(what: str, t, device: int, least: int, dtype) -> int:
    """The pointer of a contiguous tensor of that type, with that many numbers."""
    if (t.dtype is not dtype or t.numel() < least or t.get_device() != device
            or not t.is_contiguous()):
        raise ValueError(f"{what}: a contiguous {dtype} tensor on device {device}, of {least} "
                         f"numbers at least")
    return t.data_ptr()


class PagedBatch:
    """A batch over a PagedCache (dnx_paged_batch): starts [seqs + 1], lens
    [seqs] and tables [seqs][pages] as int32 tensors, which may change between
    calls (their values, in place); the number of rows, and the bounds that no
    sequence's new tokens and own keys pass. prefix_pages: the pages of the
    prefix_len keys with which every sequence begins."""

    def __init__(self, starts, lens, tables, tokens: int, max_tokens: int, max_len: int,
                 prefix_pages=None, prefix_len: int = 0):
        seqs = lens.numel()
        if tables.dim() != 2 or tables.shape[0] != seqs:
            raise ValueError("PagedBatch: tables [seqs][pages]")
        if seqs < 1 or tokens < 0 or max_tokens < 1 or max_len < 0 or prefix_len < 0:
            raise ValueError("PagedBatch: a sequence at least, and no negative numbers")
        self.starts, self.lens, self.tables, self.prefix_pages = starts, lens, tables, prefix_pages
        self.tokens, self.prefix_len = tokens, prefix_len
        self.device = d = starts.get_device()
        if d < 0:
            raise ValueError("PagedBatch: CUDA (HIP) tensors")
        self.prefix_places = 0 if prefix_pages is None else prefix_pages.numel()
        self.struct = _lib.PagedBatchStruct(
            _numbers("starts", starts, d, seqs + 1, _I32), _numbers("lens", lens, d, seqs, _I32),
            _numbers("tables", tables, d, 0, _I32),
            None if prefix_pages is None else _numbers("prefix_pages", prefix_pages, d, 0, _I32),
            tables.shape[1], prefix_len, seqs, tokens, max_tokens, max_len)
        self.ref = ctypes.addressof(self.struct)

    def check(self, cache: PagedCache) -> None:
        if self.prefix_len > self.prefix_places * cache.page:
            raise ValueError("PagedBatch: prefix_pages holds fewer pages than the prefix needs")
        if self.device != cache.device:
            raise ValueError("PagedBatch: on another device than the cache")


def paged_append(cache: PagedCache, k, v, positions, slots, rope=None, q=None, q_out=None,
                 q_norm=None, k_norm=None, eps: float = 1e-6, stream=None) -> None:
    """New tokens' keys [n][kv_heads][hd], normed and rotated, and values into
    places `slots` of the cache (dnx_paged_append); with q [n][heads][hd] also
    the queries, normed and rotated, into q_out. q, k and v may be views of one
    projection's output. A slot of -1 leaves its token out."""
    d = cache.check_device()
    shape = k.shape
    n, kv_heads, hd = shape
    ks, k1, k2 = k.stride()
    vs, v1, v2 = v.stride()
    if (kv_heads != cache.kv_heads or hd != cache.hd or v.shape != shape or k.dtype is not _F32
            or v.dtype is not _F32 or k2 != 1 or v2 != 1
            or (kv_heads != 1 and (k1 != hd or v1 != hd))):   # a lone head's stride is anything
        raise ValueError("paged_append: k and v are float32 [n][kv_heads][hd] with dense heads")
    if k.get_device() != d or v.get_device() != d:
        raise ValueError("paged_append: k and v are not on the cache's device")
    qp = qo = kw = qw = table = at = None
    qs = heads = rows = 0
    if q is not None:
        tokens, heads, dims = q.shape
        qs, q1, q2 = q.stride()
        if (tokens != n or dims != hd or q.dtype is not _F32 or q2 != 1
                or (heads != 1 and q1 != hd) or q.get_device() != d):
            raise ValueError("paged_append: q is float32 [n][heads][hd] with dense heads")
        if q_out is None:
            raise ValueError("paged_append: q needs a float32 q_out [n][heads][hd]")
        qp, qo = q.data_ptr(), _numbers("q_out", q_out, d, n * heads * hd, _F32)
    if k_norm is not None:
        kw = _numbers("k_norm", k_norm, d, hd, _F32)
    if q_norm is not None:
        qw = _numbers("q_norm", q_norm, d, hd, _F32)
    if rope is not None:
        rows, dims = rope.shape
        if dims != hd or positions is None:
            raise ValueError("paged_append: rope is float32 [positions][hd], with positions")
        table = _numbers("rope", rope, d, 0, _F32)
    if positions is not None:
        at = _numbers("positions", positions, d, n, _I32)
    if n == 1:      # a lone row's stride is anything
        qs, ks, vs = heads * hd, kv_heads * hd, kv_heads * hd
    rc = _lib.load().dnx_paged_append(
        cache.ref, qp, qs, qo, k.data_ptr(), ks, v.data_ptr(), vs, qw, kw, table, rows, at,
        _numbers("slots", slots, d, n, _I32), heads, n, eps, _on(d, stream))
    if rc:
        _check(rc, "dnx_paged_append")


def paged_attention_workspace(cache: PagedCache, batch: PagedBatch, heads: int,
                              device="cuda") -> torch.Tensor:
    """Device workspace of paged_attention for a batch of these bounds."""
    batch.check(cache)
    nbytes = int(_lib.load().dnx_paged_attention_workspace_bytes(cache.ref, batch.ref, heads))
    if nbytes < 0:
        raise RuntimeError("dnx_paged_attention_workspace_bytes refused the batch")
    return torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)


def paged_attention(cache: PagedCache, batch: PagedBatch, q, out, workspace, window: int = 0,
                    gate=None, stream=None) -> None:
    """Attention of the batch's new tokens q [tokens][heads][hd] over the shared
    prefix and each sequence's own pages, into out (dnx_paged_attention)."""
    d = cache.check_device()
    batch.check(cache)
    n, heads, hd = q.shape
    if n != batch.tokens or hd != cache.hd or q.dtype is not _F32 or out.dtype is not _F32:
        raise ValueError("paged_attention: q and out are float32 [tokens][heads][hd]")
    if out.nbytes < q.nbytes or (gate is not None and (gate.nbytes < n * heads * 4
                                                       or gate.dtype is not _F32)):
        _need("paged_attention", out=(out, q.nbytes), gate=(gate, n * heads * 4))
        raise ValueError("paged_attention: gate is float32 [tokens][heads]")
    rc = _lib.load().dnx_paged_attention(cache.ref, batch.ref, _at(q, d), _at(gate, d), _at(out, d),
                                         heads, window, _at(workspace, d), workspace.nbytes,
                                         _stream(stream))
    if rc:
        _check(rc, "dnx_paged_attention")
