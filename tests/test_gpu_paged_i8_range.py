"""dnx_paged_attention over int8 caches at the ends of the float range, against
the formula in 64 bits, with bounds that follow the digits it is made of.

Tolerances, with u = 2^-24. A query row is in multiples of 2^(e - 31), 2^e the power
of two above 1.004 times its largest value and so at most 2.008 times that value (the
rounding of 1.004 times it: 2.01): an element is off by half a unit at most, 2.01 2^-32
times the row's largest. Sums of products with codes are exact; made floats by two
roundings and scaled by four, so a score is off by 2.01 2^-32 max|q| sum|k| / sqrt(hd) +
8 u |s|, and exp2 adds 2 u. A weight times its value's scale is a multiple of 2^(e - 23)
in the same way, off by 2.01 u of the largest of its step; a step is 64 keys, so the
largest lies within 63 keys of it. The normalised weights are off by twice the scores'
error, the sums over N keys add 2 (N + 64) u of the sum of |weight v|, the gate 4 u."""

import numpy as np
import pytest
import torch
from scipy.ndimage import maximum_filter1d

from gpu_util import host
from test_gpu_paged import CASES, U
from test_gpu_paged_i8 import MORE, Batch8

pytestmark = pytest.mark.gpu


class Tight(Batch8):
    query = 2.01 * 2.0 ** -32    # an element's error in parts of the row's largest

    def take(self):
        super().take()

        def of(pages, count):
            pages = torch.from_numpy(np.asarray(pages[:-(-count // self.page)])).cuda().long()
            return (self.value_scales[pages].double().transpose(1, 2).flatten(0, 1)[:count]
                    .cpu().numpy())

        self.scales_of = [of(self.shared, self.prefix)] + [
            of(t, n) for t, n in zip(self.tables_h, self.kept_lens())]

    def expected(self, window=0, seen=None):
        want = np.zeros((self.live, self.heads, self.hd))
        room = np.zeros_like(want)
        group, t = self.heads // self.kv, 0
        q = self.q[:self.live].double().cpu().numpy()
        gate = None if self.gate is None else self.gate[:self.live].double().cpu().numpy()
        for b, (c, n) in enumerate(zip(self.counts, self.lens)):
            n_seen = min(n, self.max_len)
            k, v = (np.concatenate([f.cpu().numpy(), o.cpu().numpy()[:n_seen]])
                    for f, o in zip(self.first_kv, self.own_kv[b]))
            unit = np.concatenate([self.scales_of[0], self.scales_of[1 + b][:n_seen]])
            there = np.array([seen is None or seen(b, j) for j in range(len(k))], bool)
            for i in range(c):
                p = self.prefix + n - c + i
                j = np.arange(len(k))
                ok = there & (j <= p) & ((j > p - window) if window else True)
                for h in range(self.heads) if ok.any() else ():
                    kk, vv, vs = k[ok, h // group], v[ok, h // group], unit[ok, h // group]
                    s = kk @ q[t, h] / np.sqrt(self.hd)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    e = (self.query * np.abs(q[t, h]).max() * np.abs(kk).sum(1) / np.sqrt(self.hd)
                         + 8 * U * np.abs(s)).max() + 2 * U
                    of_step = maximum_filter1d(w * vs, 127, mode="constant")
                    codes = np.abs(vv) / np.where(vs > 0, vs, 1)[:, None]
                    want[t, h] = w @ vv
                    room[t, h] = ((2 * e + 2 * (len(kk) + 64) * U) * (w @ np.abs(vv))
                                  + 2.01 * U * of_step @ codes)
                    if gate is not None:
                        g = 1 / (1 + np.exp(-gate[t, h]))
                        room[t, h] = (room[t, h] + 4 * U * np.abs(want[t, h])) * g
                        want[t, h] *= g
                t += 1
        return want, room


SHAPES = [([1, 3], [200, 90], 70), ([150], [200], 0), ([40, 1], [90, 300], 777), ([1], [1], 0)]


def batch(seed, shape, hd, **more):
    counts, lens, prefix = shape
    return Tight(seed, counts, lens, prefix, 8, 2, hd, 32, **more)


def times(t, exponents):
    """t times powers of two, with float32's own rounding where that is subnormal."""
    x = t.double().cpu().numpy() * np.exp2(np.asarray(exponents, np.float64))
    t.copy_(torch.from_numpy(x.astype(np.float32)))


@pytest.mark.parametrize("case", range(len(CASES + MORE)))
def test_attention(gpu_ready, case):
    counts, lens, prefix, heads, kv, hd, page = (CASES + MORE)[case]
    Tight(case, counts, lens, prefix, heads, kv, hd, page, pad=case % 3, gate=case % 2 == 1).check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_queries_of_nearly_nothing(gpu_ready, shape, hd):
    """Rows down to the last subnormals, of one size and of every size beside each
    other: the plain mean of what is seen, also in steps with masked keys."""
    for by in (-33, -60, -100, -118, -126, -130, -140, -148, -149, -160):
        b = batch(50, SHAPES[shape], hd)
        times(b.q, by)
        b.check()
        b.check(50)
    b = batch(51, SHAPES[shape], hd, gate=True)
    rng = np.random.default_rng(hd)
    rows = tuple(b.q.shape[:2])
    times(b.q, rng.integers(-155, 4, rows)[..., None])
    b.q[rng.random(rows) < 0.1] = 0.0
    b.check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_small_queries_on_large_keys_and_the_reverse(gpu_ready, shape, hd):
    """Scores of ordinary size whose factors are not."""
    for by in (20, 31, 33, 80, 100, 110, -20, -60, -90, -115):
        b = batch(52, SHAPES[shape], hd)
        times(b.key_scales, by)
        times(b.q, -by)
        b.take()
        b.check()
    b = batch(53, SHAPES[shape], hd)
    rng = np.random.default_rng(hd)
    rows = tuple(b.q.shape[:2])
    times(b.key_scales, 105)
    times(b.q, rng.integers(-120, -98, rows)[..., None])
    b.take()
    b.check()


def test_subnormal_queries_on_the_largest_keys(gpu_ready):
    """Rows of a few bits, whose scores count nevertheless."""
    for shape in SHAPES:
        for by, more in ((-130, 118), (-140, 118)):
            b = batch(54, shape, 128)
            times(b.q, by)
            times(b.key_scales, more)
            b.take()
            b.check()
            q = host(b.q)
            assert (np.abs(q).max() < 2.0 ** -120) and (q != 0).any()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_one_large_query_channel(gpu_ready, shape, hd):
    """A channel that is large in the queries and small in the keys, as models have
    them: the others keep their bits."""
    for by in (30.0, 300.0, 3000.0, 1e5, 1e6):
        b = batch(55, SHAPES[shape], hd, gate=by > 1000)
        rng = np.random.default_rng(int(by))
        at = int(rng.integers(hd))
        b.q[..., at] *= by
        b.keys[..., at] = (b.keys[..., at].float() / by).round().to(torch.int8)
        b.take()
        b.check()
        b.check(70)
