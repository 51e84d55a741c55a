"""dnx_sample where |l / T| is so large that neighbouring floats lie many bins
apart: requests with top-k and top-p together, whose cut by weight lies in a
bin that the bins' own weights cannot tell. Tokens as in test_gpu_sample.py:
equal to those of the definition in 64 bits, both of two where a border lies
within 1e-9 (each weight is off by half of 2^-43 of the largest, so that a sum of
up to 2^20 of them is off by 2^-24 of it at most and by 1e-11 for the few that
weigh anything here)."""

import numpy as np
import pytest
import torch

from dianoia_amd import device as D
from test_gpu_sample import Rows, logits_of

pytestmark = pytest.mark.gpu


def steps_below(top, n):
    """top and the n - 1 floats below it."""
    out = [np.float32(top)]
    for _ in range(n - 1):
        out.append(np.nextafter(out[-1], np.float32(-np.inf)))
    return np.array(out, np.float32)


def near_rows(rng, rows, vocab, tops, count):
    """Rows of a low floor with `count` tokens from tops[row] down, one float each."""
    l = np.full((rows, vocab), -1e30, np.float32)
    at = np.array([rng.permutation(vocab)[:count] for _ in range(rows)])
    for r in range(rows):
        l[r, at[r]] = rng.permutation(steps_below(tops[r % len(tops)], count))
    return l


# |top / T| from 2^20 to 2^30: with t = a float's step at top, times one to three, so
# that neighbours weigh e^-1 to e^-1/3 of each other.
TOPS = [1.0, 20.0, -20.0, 1000.0, 8388612.0, -7.5e6]


@pytest.mark.parametrize("vocab", [100, 3000, 40000, 151936])
@pytest.mark.parametrize("rows", [6, 300])
def test_both_filters_on_neighbouring_floats(gpu_ready, vocab, rows):
    if rows > 6 and vocab > 3000:
        rows = 24
    rng = np.random.default_rng(vocab + rows)
    for count in (3, 5, 40):
        l = near_rows(rng, rows, vocab, TOPS, count)
        step = np.spacing(np.abs(l.max(1)))
        t = (step * rng.choice([1.0, 1.7, 3.0], rows)).astype(np.float32)
        k = rng.choice([2, 3, 4, 5, 39], rows)
        p = rng.choice([0.3, 0.5, 0.7, 0.9, 0.99], rows)
        for u in (0.0, 0.5, 0.9, 0.999):
            Rows(l, u, t=t, k=k, p=p).check()
        Rows(l, rng.random(rows), t=t, k=k, p=p, low=0.2).check()
        Rows(l, rng.random(rows), t=t, p=p).check()
        Rows(l, rng.random(rows), t=t, k=k).check()


def test_three_floats_after_a_row_of_many(gpu_ready):
    """The cut by weight keeps two of three tokens, in calls whose other rows have
    long lists of near tokens; one launch and four."""
    rng = np.random.default_rng(1)
    for rows, vocab in ((256, 4000), (300, 4000), (64, 50000)):
        l = (0.05 * rng.standard_normal((rows, vocab))).astype(np.float32)
        t, k, p = np.ones(rows, np.float32), np.full(rows, vocab // 3), np.full(rows, 0.5)
        few = np.arange(rows // 2, rows)
        l[few] = -1e30
        l[few[:, None], [3, 40, 77]] = np.float32([8388612, 8388611, 8388610])
        l[few[1::2, None], [3, 40, 77]] = steps_below(20.0, 3)
        t[few[1::2]] = 2e-6
        k[few], p[few] = 3, 0.7
        r = Rows(l, 0.9, t=t, k=k, p=p)
        for _ in range(3):
            assert (r.run()[few] == 40).all()
        r.check()


@pytest.mark.parametrize("t", [1e-3, 1e-5, 1e-7, 1e-12, 1e-38, 1e-45])
def test_temperatures_of_nearly_nothing(gpu_ready, t):
    """Ordinary logits, with ties for the largest: |l / T| up to infinity."""
    rng = np.random.default_rng(2)
    for vocab in (1000, 40000):
        l = logits_of(rng, 12, vocab)
        for r in range(0, 12, 2):
            l[r, rng.permutation(vocab)[:4]] = l[r].max()
        for par in (dict(k=3, p=0.7), dict(k=50, p=0.4, low=0.1), dict(p=0.9), dict(k=2)):
            Rows(l, rng.random(12), t=np.float32(t), **par).check()


@pytest.mark.parametrize("rows,vocab", [(32, 32003), (114, 9000), (257, 32003), (54, 151936), (9, 128000)])
def test_fewer_rows_and_tokens_in_the_same_workspace(gpu_ready, rows, vocab):
    """A server's workspace is that of its largest batch; nothing behind it is written."""
    rng = np.random.default_rng(rows)
    n = D.sample_workspace(rows, vocab).nbytes
    memory = torch.full((n + 4096,), 0xff, dtype=torch.uint8, device="cuda")
    l = logits_of(rng, rows, vocab)
    for fewer in {rows, rows - 1, rows // 2, 1}:
        for tokens in {vocab, vocab - 1, vocab // 2 + 3, 8193, 700}:
            r = Rows(l[:fewer, :tokens], rng.random(fewer), t=0.8, k=rng.choice([0, 40], fewer), p=0.9)
            out = torch.full((fewer,), -9, dtype=torch.int32, device="cuda")
            t, k, p, _ = (None if x is None else torch.from_numpy(x).cuda() for x in r.par)
            D.sample(r.logits, torch.from_numpy(r.u).cuda(), out, memory[:n], temperature=t, top_k=k, top_p=p)
            assert (out.cpu().numpy() == r.run()).all()
    assert bool((memory[n:] == 0xff).all())
