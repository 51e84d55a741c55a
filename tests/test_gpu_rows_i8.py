"""int8 rows with one scale each (dnx_quantize_i8r*, dnx_rms_norm_i8r) and
their product (dnx_gemm_i8r), against the formulas in 64 bits.

Tolerances. A code is the nearest whole number to 127 y / max|y|, halves away
from zero: for the rows as they are 254 |x| - (2 k + 1) max is exact in 64
bits, so codes must be equal, ties too; for the norm the kernel's 64-bit
factor is off by a few 2^-53, which no seeded value here lies that near to a
border. A scale is one rounding of a 64-bit value: 2^-24. A product is the
exact sum rounded once, the scales' product once, their product once: 3 2^-24
(and its square)."""

import numpy as np
import pytest
import torch

from dianoia_amd import device as D
from gpu_util import bits, dev, host
from test_gemm_i8r_route import MORE as MORE_TILES, SHAPES as TILES

U = 2.0 ** -24
EPS = 1e-6


def round_half_away(t):
    return np.sign(t) * np.floor(np.abs(t) + 0.5)


def reference(y):
    """Codes and scales of float64 rows."""
    top = np.abs(y).max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        code = np.where(top > 0, round_half_away(127.0 * y / top), 0.0)
    return code.astype(np.int8), top[:, 0] / 127.0


def outputs(rows, pad):
    """Sentinels behind the last row show what is written past it."""
    return (torch.full((rows + 1, pad), 77, dtype=torch.int8, device="cuda"),
            torch.full((rows + 1,), 7.5, device="cuda"))


def check(qs, scales, code, scale, rows, cols, pad):
    q, s = host(qs), host(scales)
    assert np.array_equal(q[:rows, :cols], code)
    assert (q[:rows, cols:] == 0).all()
    assert (q[rows] == 77).all() and s[rows] == 7.5
    assert (np.abs(s[:rows] - scale) <= U * scale * (1 + 1e-7)).all()


SHAPES = [(1, 4, 32), (1, 32, 32), (3, 260, 288), (17, 1000, 1024), (5, 4096, 4096),
          (2, 4100, 4128), (300, 1152, 1152), (2, 12292, 12320), (1, 20000, 20000),
          (2, 65536, 65536)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,pad", SHAPES)
def test_quantize(gpu_ready, rows, cols, pad):
    rng = np.random.default_rng(rows * cols)
    x = (rng.standard_normal((rows, cols)) * 3).astype(np.float32)
    qs, scales = outputs(rows, pad)
    D.quantize_i8r(dev(x), qs, scales, rows, cols, pad)
    check(qs, scales, *reference(x.astype(np.float64)), rows, cols, pad)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,pad", SHAPES)
def test_quantize_bf16(gpu_ready, rows, cols, pad):
    """Eight significant bits: many values lie on the border of two codes."""
    rng = np.random.default_rng(rows + cols)
    w = torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32) * 0.02).bfloat16()
    qs, scales = outputs(rows, pad)
    D.quantize_i8r_bf16(w.cuda(), qs, scales, rows, cols, pad)
    check(qs, scales, *reference(w.double().numpy()), rows, cols, pad)


@pytest.mark.gpu
def test_quantize_ties(gpu_ready):
    """Every tie of a row whose largest value is 381: x = 1.5 (2 k + 1)."""
    x = np.zeros((2, 256), np.float32)
    x[0, :127] = 1.5 * (2 * np.arange(127) + 1)
    x[0, 127] = 381.0
    x[0, 128:255] = -x[0, :127]
    x[1] = -np.nextafter(x[0], np.float32(0))
    x[1, 127] = 381.0
    qs, scales = outputs(2, 256)
    D.quantize_i8r(dev(x), qs, scales, 2, 256, 256)
    q = host(qs)
    assert np.array_equal(q[0, :127], np.arange(127) + 1)
    assert np.array_equal(q[0, 128:255], -np.arange(127) - 1)
    assert np.array_equal(q[1, :127], -np.arange(127))
    check(qs, scales, *reference(x.astype(np.float64)), 2, 256, 256)


@pytest.mark.gpu
def test_extremes(gpu_ready):
    """Zero rows, the smallest and largest floats, infinities and NaN."""
    x = np.zeros((7, 64), np.float32)
    x[1, 3] = 1e-45
    x[2, :2] = 3.4e38, -3.4e38
    x[3, 5] = -0.0
    x[4, :3] = 1.0, np.inf, -2.0
    x[5, :3] = 1.0, np.nan, -2.0
    x[6, :3] = 1.0, 0.5, -2.0
    qs, scales = outputs(7, 64)
    D.quantize_i8r(dev(x), qs, scales, 7, 64, 64)
    q, s = host(qs), host(scales)
    assert (q[[0, 3]] == 0).all() and (s[[0, 3]] == 0).all()
    assert q[1, 3] == 127 and s[1] == 0.0            # the scale is below the smallest float
    assert q[2, 0] == 127 and q[2, 1] == -127
    assert np.isnan(s[4]) and np.isnan(s[5])
    assert q[6, 0] == 64 and q[6, 1] == 32 and q[6, 2] == -127
    w = np.ones(64, np.float32)
    D.rms_norm_i8r(dev(x), dev(w), qs, scales, 7, 64, 64, EPS)
    q, s = host(qs), host(scales)
    assert (q[[0, 3]] == 0).all() and (s[[0, 3]] == 0).all()
    assert np.isnan(s[4]) and np.isnan(s[5])
    assert q[6, 0] == 64 and q[6, 2] == -127


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("rows", [3, 600])
def test_norm_weight_without_a_code(gpu_ready, rows, bad):
    """An infinity or NaN in the weight reaches every row's scale."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((rows, 96)).astype(np.float32)
    w = np.ones(96, np.float32)
    w[50] = bad
    qs, scales = outputs(rows, 96)
    D.rms_norm_i8r(dev(x), dev(w), qs, scales, rows, 96, 96, EPS)
    assert np.isnan(host(scales)[:rows]).all() and (host(qs)[:rows] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [16384, 16388, 40000])
@pytest.mark.parametrize("at", [0, -1])
def test_long_norm_rows_without_a_code(gpu_ready, cols, at):
    """Rows about the length from which they are read twice."""
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((4, cols)).astype(np.float32)
    x[0], x[1, at], x[2, at] = 0.0, np.nan, -np.inf
    w = np.ones(cols, np.float32)
    pad = -(-cols // 32) * 32
    qs, scales = outputs(4, pad)
    D.rms_norm_i8r(dev(x), dev(w), qs, scales, 4, cols, pad, EPS)
    q, s = host(qs), host(scales)
    assert (q[:3] == 0).all() and s[0] == 0 and np.isnan(s[1]) and np.isnan(s[2])
    assert np.abs(q[3].astype(int)).max() == 127 and np.isfinite(s[3])
    w[at] = np.inf
    D.rms_norm_i8r(dev(x), dev(w), qs, scales, 4, cols, pad, EPS)
    assert np.isnan(host(scales)[:4]).all() and (host(qs)[:4] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,pad", SHAPES + [(600, 260, 288), (513, 4096, 4096),
                                                    (700, 8196, 8224)])
@pytest.mark.parametrize("add", [False, True])
def test_norm(gpu_ready, rows, cols, pad, add):
    rng = np.random.default_rng(rows * 7 + cols + add)
    x = rng.standard_normal((rows, cols)).astype(np.float32)
    m = rng.standard_normal((rows, cols)).astype(np.float32)
    w = (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    total = x + m if add else x
    s = total.astype(np.float64)
    r = 1.0 / np.sqrt((s * s).mean(1, keepdims=True) + np.float64(np.float32(EPS)))
    code, scale = reference(w.astype(np.float64) * s)
    qs, scales = outputs(rows, pad)
    xd = dev(x)
    x_out = torch.full((rows + 1, cols), 5.0, device="cuda") if add else None
    D.rms_norm_i8r(xd, dev(w), qs, scales, rows, cols, pad, EPS, m=dev(m) if add else None,
                   x_out=x_out)
    check(qs, scales, code, scale * r[:, 0], rows, cols, pad)
    assert np.array_equal(bits(host(xd)), bits(x))
    if add:
        out = host(x_out)
        assert np.array_equal(bits(out[:rows]), bits(total)) and (out[rows] == 5.0).all()
        # In place, into x and into m: the same.
        for into in ("x", "m"):
            xd, md = dev(x), dev(m)
            q2, s2 = outputs(rows, pad)
            D.rms_norm_i8r(xd, dev(w), q2, s2, rows, cols, pad, EPS, m=md,
                           x_out=xd if into == "x" else md)
            assert np.array_equal(bits(host(xd if into == "x" else md)), bits(total))
            assert torch.equal(q2, qs) and torch.equal(s2, scales)


PRODUCTS = [(1, 1, 32), (1, 33, 64), (5, 31, 96), (13, 1000, 2048), (16, 64, 4096),
            (17, 4099, 1120), (31, 200, 32), (64, 300, 320), (65, 129, 4096), (100, 2050, 1152),
            (128, 1024, 1024), (255, 257, 544), (257, 770, 2080), (600, 515, 160),
            (1024, 4304, 1152), (1, 9000, 4096), (3, 128, 131040)]


# Two tiles of rows a workgroup: whole, and a last one that is partly there.
PRODUCTS += [(5, 8192, 64), (16, 8161, 96), (9, 4113, 2080), (13, 33001, 160)]


@pytest.mark.gpu
@pytest.mark.parametrize("n,rows,cols", PRODUCTS)
def test_product(gpu_ready, n, rows, cols):
    rng = np.random.default_rng(n + rows + cols)
    w = rng.integers(-128, 128, (rows, cols), dtype=np.int8)
    x = rng.integers(-128, 128, (n, cols), dtype=np.int8)
    ws = (rng.random(rows) * 1e-3).astype(np.float32)
    xs = (rng.random(n) * 1e-2).astype(np.float32)
    y = torch.full((n * rows + 64,), 3.5, device="cuda")
    D.gemm_i8r(dev(w), dev(ws), dev(x), dev(xs), y, rows, cols, n)
    got = host(y)
    exact = x.astype(np.float64) @ w.astype(np.float64).T
    exact = exact * xs[:, None].astype(np.float64) * ws.astype(np.float64)
    assert (np.abs(got[:n * rows].reshape(n, rows) - exact) <= 3 * U * (1 + 2 * U) * np.abs(exact)).all()
    assert (got[n * rows:] == 3.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", TILES + MORE_TILES)
@pytest.mark.parametrize("shift", [0, 1])
def test_product_every_tile(gpu_ready, shape, shift):
    """Each tile kernel of the route, at odd sizes and at rows of a multiple of
    4, the outputs on 16 bytes or not. Sums below 2^53 are exact in float64."""
    n, rows, cols = shape
    for rows in (rows, rows // 4 * 4):
        print(f"product {n} x {rows} x {cols}", flush=True)
        g = torch.Generator(device="cuda").manual_seed(n)
        w, x = (torch.randint(-128, 128, (r, cols), device="cuda", generator=g).to(torch.int8)
                for r in (rows, n))
        ws, xs = (torch.rand(r, device="cuda", generator=g) + 0.5 for r in (rows, n))
        y = torch.full((shift + n * rows + 64,), 3.5, device="cuda")
        D.gemm_i8r(w, ws, x, xs, y[shift:], rows, cols, n)
        exact = (x.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
        got = y[shift:shift + n * rows].view(n, rows).double()
        assert ((got - exact).abs() <= 3 * U * (1 + 2 * U) * exact.abs()).all()
        assert (y[:shift] == 3.5).all() and (y[shift + n * rows:] == 3.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [131040, 4096])
def test_product_largest_sums(gpu_ready, cols):
    """Every code at the end of its range: the sum that comes nearest to 2^31."""
    n, rows = 2, 40
    w = np.full((rows, cols), -128, np.int8)
    x = np.full((n, cols), -128, np.int8)
    x[1] = 127
    one = np.ones(rows, np.float32)
    y = torch.empty(n, rows, device="cuda")
    D.gemm_i8r(dev(w), dev(one), dev(x), dev(one[:n]), y, rows, cols, n)
    got = host(y).astype(np.float64)
    for t, v in ((0, 16384.0 * cols), (1, -16256.0 * cols)):
        assert (np.abs(got[t] - v) <= U * abs(v)).all()


@pytest.mark.gpu
def test_product_scales_pass_through(gpu_ready):
    """Zero, infinite and NaN scales: that token's or row's outputs alone."""
    w, x = np.ones((64, 64), np.int8), np.ones((3, 64), np.int8)
    xs = np.array([1.0, np.nan, 0.0], np.float32)
    ws = np.ones(64, np.float32)
    ws[5], ws[6] = np.inf, np.nan
    y = torch.empty(3, 64, device="cuda")
    D.gemm_i8r(dev(w), dev(ws), dev(x), dev(xs), y, 64, 64, 3)
    got = host(y)
    assert np.isnan(got[1]).all() and np.isinf(got[0, 5]) and np.isnan(got[0, 6])
    assert np.isnan(got[2, 5]) and (np.delete(got[0], [5, 6]) == 64).all()
    assert (np.delete(got[2], [5, 6]) == 0).all()


@pytest.mark.gpu
def test_rows_then_product_on_a_stream_and_in_a_graph(gpu_ready):
    """The norm's rows into the product as a decode step runs them: on a side
    stream, and captured and replayed over changing inputs."""
    n, rows, cols = 9, 770, 1152
    rng = np.random.default_rng(5)
    w16 = torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32) * 0.05).bfloat16().cuda()
    norm = dev((1 + 0.1 * rng.standard_normal(cols)).astype(np.float32))
    wq = torch.empty(rows, cols, dtype=torch.int8, device="cuda")
    ws, xs = torch.empty(rows, device="cuda"), torch.empty(n, device="cuda")
    xq = torch.empty(n, cols, dtype=torch.int8, device="cuda")
    D.quantize_i8r_bf16(w16, wq, ws, rows, cols, cols)
    x, m = torch.empty(n, cols, device="cuda"), torch.empty(n, cols, device="cuda")
    y = torch.empty(n, rows, device="cuda")

    def step(stream=None):
        D.rms_norm_i8r(x, norm, xq, xs, n, cols, cols, EPS, m=m, x_out=x, stream=stream)
        D.gemm_i8r(wq, ws, xq, xs, y, rows, cols, n, stream=stream)

    def fill(k):
        g = torch.Generator(device="cuda").manual_seed(k)
        x.copy_(torch.randn(n, cols, device="cuda", generator=g))
        m.copy_(torch.randn(n, cols, device="cuda", generator=g))

    want = []
    for k in range(4):
        fill(k)
        step()
        want.append((y.clone(), x.clone()))
    side = torch.cuda.Stream()
    fill(0)
    side.wait_stream(torch.cuda.current_stream())
    step(side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, want[0][0]) and torch.equal(x, want[0][1])
    fill(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in (1, 2, 3, 1):
        fill(k)
        y.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[k][0]) and torch.equal(x, want[k][1])
    # The chain against 64 bits: |y| is off by what the two roundings to 8
    # bits (half a step each, of the row's largest / 127) can amount to.
    s = want[2][1].double()
    h = s * torch.rsqrt((s * s).mean(1, keepdim=True) + EPS) * norm.double()
    wd = w16.double()
    exact = h @ wd.t()
    hx, wx = h.abs().amax(1, keepdim=True) / 254, wd.abs().amax(1) / 254
    room = hx * (wd.abs().sum(1) + cols * wx) + h.abs().sum(1, keepdim=True) * wx
    assert ((want[2][0] - exact).abs() <= room * (1 + 1e-5)).all()


def test_refusals():
    """Refused before anything is launched (no GPU is needed for these)."""
    from dianoia_amd import _lib
    lib = _lib.load()
    a = 4096   # a pointer that no refused call reads
    quant = lambda **k: lib.dnx_quantize_i8r(*{**dict(x=a, q=a, s=a, rows=2, cols=64, pad=64, st=None), **k}.values())
    for bad in (dict(cols=0), dict(cols=63), dict(cols=65540, pad=65568), dict(pad=32), dict(pad=70),
                dict(rows=-1), dict(rows=1 << 31), dict(x=a + 4), dict(q=a + 8), dict(s=a + 2),
                dict(x=None), dict(q=None), dict(s=None)):
        assert quant(**bad) == -1, bad
    assert quant(rows=0) == 0
    norm = lambda **k: lib.dnx_rms_norm_i8r(*{**dict(x=a, m=a, o=a, w=a, q=a, s=a, rows=2, cols=64, pad=64, eps=EPS, st=None), **k}.values())
    for bad in (dict(m=None), dict(o=None), dict(w=None), dict(w=a + 4), dict(m=a + 4), dict(o=a + 8)):
        assert norm(**bad) == -1, bad
    gemm = lambda **k: lib.dnx_gemm_i8r(*{**dict(w=a, ws=a, x=a, xs=a, y=a, rows=8, cols=64, n=2, st=None), **k}.values())
    for bad in (dict(cols=48), dict(cols=0), dict(cols=131072), dict(rows=0), dict(rows=1 << 31), dict(n=-1),
                dict(n=1 << 31), dict(w=a + 8), dict(x=a + 4), dict(y=a + 2), dict(ws=a + 1), dict(w=None),
                dict(xs=None)):
        assert gemm(**bad) == -1, bad
    assert gemm(n=0) == 0
    t = torch.zeros(64)
    with pytest.raises(ValueError):   # smaller than the shape needs
        D.quantize_i8r(t, t, t, 2, 64, 64)
    with pytest.raises(ValueError):
        D.gemm_i8r(t, t, t, t, t, 8, 64, 2)
    with pytest.raises(ValueError):   # not in HBM
        D.quantize_i8r(t, t, t, 1, 64, 64)


def test_types_are_refused():
    """A tensor large enough, but of another type than the kernel reads or
    writes: refused before anything is launched, by its name."""
    h, d = torch.zeros(64, 64).half(), torch.zeros(64, 64).double()
    b, q, u = h.bfloat16(), torch.zeros(64, 64, dtype=torch.int8), torch.zeros(64, 64, dtype=torch.uint8)
    s, s64 = torch.zeros(64), torch.zeros(64).double()
    for f in (D.quantize_i8r, D.quantize_i8r_bf16):
        x = torch.zeros(64, 64, dtype=torch.float32 if f is D.quantize_i8r else torch.bfloat16)
        for args, what in (((h if f is D.quantize_i8r_bf16 else d, q, s), "x is"), ((x, u, s), "qs is"),
                           ((x, q, s64), "scales is"), ((d, q, s), "x is")):
            with pytest.raises(ValueError, match=what):
                f(*args, 64, 64, 64)
        with pytest.raises(ValueError, match="CUDA"):      # of its types, but not in HBM
            f(x, q, s, 64, 64, 64)
    with pytest.raises(ValueError, match="CUDA"):          # bf16 bits
        D.quantize_i8r_bf16(b.view(torch.int16), q, s, 64, 64, 64)
    x = torch.zeros(64, 64)
    norm = dict(x=x, w=s, qs=q, scales=s, m=x, x_out=x)
    for name, bad in (("x", d), ("w", s64), ("qs", u), ("scales", s64), ("m", d), ("x_out", d)):
        with pytest.raises(ValueError, match=f"{name} is"):
            D.rms_norm_i8r(**{**norm, name: bad}, rows=64, cols=64, cols_pad=64, eps=EPS)
    product = dict(w=q, w_scale=s, x=q, x_scale=s, y=x)
    for name, bad in (("w", u), ("w_scale", s64), ("x", x), ("x_scale", s64), ("y", d)):
        with pytest.raises(ValueError, match=f"{name} is"):
            D.gemm_i8r(**{**product, name: bad}, rows=64, cols=64, n=64)
