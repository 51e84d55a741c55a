"""dnx_sample against the definition in 64 bits. Tokens are whole numbers and
have to be equal, but where u times the sum, or a cut by weight, lies within
1e-9 of the border between two tokens: there either is right. (A weight is
rounded to 2^-44 of the largest, and of a cut by top_p a sum of weights to 2^-35
of each: for up to 2^20 tokens below 1e-10 of the sums.)"""

import numpy as np
import pytest
import torch

from dianoia_amd import device as D

pytestmark = pytest.mark.gpu

NEAR = 1e-9


def answers(l, u, t, k, p, low):
    """Every token that the definition allows, borders as near as NEAR both ways."""
    l = l.astype(np.float64).copy()
    l[np.isnan(l)] = -np.inf
    if not (l > -np.inf).any():
        return {-1}
    order = np.lexsort((np.arange(l.size), -l))
    if not t > 0:
        return {int(order[0])}
    order = order[l[order] > -np.inf]
    if 0 < k < l.size:
        order = order[:k]
    with np.errstate(invalid="ignore"):
        w = np.where(l[order] == l[order[0]], 1.0, np.exp((l[order] - l[order[0]]) / t))
    if l[order[0]] == np.inf:
        w = (l[order] == np.inf).astype(np.float64)
    sizes = {w.size}
    if p < 1:
        s = np.cumsum(w)
        sizes = {max(1, int(np.searchsorted(s, max(p, 0) * s[-1] * (1 + e))) + 1) for e in (-NEAR, 0, NEAR)}
    ends = set()
    for n in sizes:
        if low > 0:
            ends |= {max(1, int((w[:n] >= min(low, 1) * (1 + e)).sum())) for e in (-NEAR, 0, NEAR)}
        else:
            ends.add(min(n, w.size))
    found = set()
    for n in ends:
        by_index = np.argsort(order[:n])
        at, s = order[:n][by_index], np.cumsum(w[:n][by_index])
        for e in (-NEAR, 0, NEAR):
            x = min(max(u if u == u else 0, 0), 1) * s[-1] + e * s[-1]
            i = int(np.searchsorted(s, max(x, 0), side="right"))
            if i >= n:                            # the last one that weighs something
                i = int(np.searchsorted(s, s[-1], side="left"))
            found.add(int(at[i]))
    return found


class Rows:
    def __init__(self, logits, u, t=None, k=None, p=None, low=None):
        self.l = np.asarray(logits, np.float32)
        n = self.l.shape[0]
        self.u = np.broadcast_to(np.asarray(u, np.float32), n).copy()
        self.par = [None if x is None else np.broadcast_to(np.asarray(x, d), n).copy()
                    for x, d in ((t, np.float32), (k, np.int32), (p, np.float32), (low, np.float32))]
        self.logits = torch.from_numpy(self.l).cuda()

    def run(self, logits=None):
        rows, vocab = self.l.shape
        out = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
        ws = D.sample_workspace(rows, vocab)
        ws.fill_(0xff)
        t, k, p, low = (None if x is None else torch.from_numpy(x).cuda() for x in self.par)
        D.sample(self.logits if logits is None else logits, torch.from_numpy(self.u).cuda(), out, ws,
                 temperature=t, top_k=k, top_p=p, min_p=low)
        return out.cpu().numpy()

    def check(self):
        got = self.run()
        none = (1.0, 0, 1.0, 0.0)
        for i in range(len(self.l)):
            par = [d if x is None else x[i] for x, d in zip(self.par, none)]
            want = answers(self.l[i], self.u[i], *par)
            assert int(got[i]) in want, (i, int(got[i]), want, par, self.u[i])
        return got


def logits_of(rng, rows, vocab, floor=2.0, some=20):
    l = floor * rng.standard_normal((rows, vocab))
    for r in l:
        r[rng.integers(0, vocab, some)] += 6 + 2.5 * rng.standard_normal(some)
    return l.astype(np.float32)


VOCABS = [1, 2, 63, 64, 65, 255, 1000, 4095, 4096, 4097, 8191, 8193, 32003, 65536, 151936]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("filters", ["none", "k", "p", "min", "all", "greedy"])
def test_sample(gpu_ready, vocab, filters):
    rng = np.random.default_rng(vocab)
    rows = 13 if vocab < 60000 else 4
    l = logits_of(rng, rows, vocab)
    u = rng.random(rows).astype(np.float32)
    t = rng.choice([0.3, 0.7, 1.0, 1.5], rows)
    k = rng.choice([1, 2, 20, 50, 1000, vocab - 1, vocab, vocab + 5, 0, -3], rows)
    p = rng.choice([0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 1.0], rows)
    low = rng.choice([0.0, 0.001, 0.05, 0.3, 1.0], rows)
    par = {"none": {}, "k": dict(t=t, k=k), "p": dict(t=t, p=p), "min": dict(t=t, low=low),
           "all": dict(t=t, k=k, p=p, low=low), "greedy": dict(t=0.0, k=k, p=p, low=low)}[filters]
    Rows(l, u, **par).check()


@pytest.mark.parametrize("vocab", [5, 300, 5000, 100000])
@pytest.mark.parametrize("what", ["equal", "two", "steps", "halves", "near"])
def test_ties(gpu_ready, vocab, what):
    """Equal logits: the lowest index first, in every filter."""
    rng = np.random.default_rng(vocab)
    rows = 12
    l = {"equal": np.full((rows, vocab), -3.5),
         "two": rng.integers(0, 2, (rows, vocab)) * 1.0,
         "steps": rng.integers(0, 9, (rows, vocab)) * 0.5,
         "halves": np.where(np.arange(vocab) % 2 == 0, 0.0, -0.0) * np.ones((rows, 1)),
         "near": 5.0 + rng.integers(0, 50, (rows, vocab)) * 2.0 ** -21}[what].astype(np.float32)
    k = np.array([0, 1, 2, 3, 7, vocab // 2, vocab - 1, 40, 64, 300, 2049, 1])
    p = np.array([1, 0.5, 0.1, 0.9, 1, 1, 0.25, 0.0, 0.999, 0.3, 0.6, 1.0])
    Rows(l, rng.random(rows), t=1.0, k=k).check()
    Rows(l, rng.random(rows), t=0.7, p=p).check()
    Rows(l, rng.random(rows), t=1.0, k=k, p=p, low=0.2).check()
    greedy = Rows(l, 0.5, t=0.0).check()
    assert (greedy == l.argmax(1)).all()


def test_borders_of_u(gpu_ready):
    rng = np.random.default_rng(0)
    for vocab in (3, 5000):
        l = logits_of(rng, 7, vocab)
        u = np.array([0.0, np.nextafter(np.float32(1), np.float32(0)), 1.0, -1.0, np.nan, np.inf, 2.0])
        for par in ({}, dict(k=3), dict(p=0.9)):
            Rows(l, u, **par).check()
    l = np.zeros((8, 4), np.float32)              # quarters: the border is the next token's
    assert Rows(l, np.arange(8) / 8).check().tolist() == [0, 0, 1, 1, 2, 2, 3, 3]


@pytest.mark.parametrize("vocab", [4, 700, 40000])
def test_special_logits(gpu_ready, vocab):
    """-inf (a mask), the lowest float, NaN, +inf, and rows of nothing."""
    rng = np.random.default_rng(vocab)
    l = logits_of(rng, 12, vocab)
    l[0] = -np.inf
    l[1] = np.nan
    l[2, ::2], l[2, 1::2] = np.nan, -np.inf
    l[3, 1:] = -np.inf
    l[4, :-1] = np.finfo(np.float32).min
    l[5] = np.finfo(np.float32).min               # a mask's value everywhere: all equal
    l[6, vocab // 2] = np.inf
    l[7, [0, vocab - 1]] = np.inf
    l[8, ::3] = np.nan
    l[9, rng.random(vocab) < 0.9] = -np.inf
    l[10, 0], l[10, 1:] = np.finfo(np.float32).max, np.finfo(np.float32).min
    u = rng.random(12)
    for par in ({}, dict(t=0.0), dict(k=2), dict(p=0.8), dict(low=0.1), dict(t=1e-30), dict(t=1e30),
                dict(t=np.inf), dict(t=np.nan), dict(t=-1.0), dict(p=np.nan, low=np.nan),
                dict(p=-1.0), dict(low=2.0), dict(k=vocab - 1, p=0.99, low=1e-6)):
        got = Rows(l, u, **par).check()
        assert got[0] == got[1] == got[2] == -1 and got[3] == 0


def test_peaked_and_flat(gpu_ready):
    """One token with nearly all the weight and a long tail; all of nearly equal
    weight; temperatures that make one of the other."""
    rng = np.random.default_rng(5)
    l = rng.standard_normal((10, 50000)).astype(np.float32)
    l[:, 777] += 25
    u = np.array([0, 0.1, 0.5, 0.9, 0.99, 0.999, 0.9999, 0.99999, 0.999999, 0.9999999])
    for t in (0.1, 1.0, 3.0, 30.0, 1e6):
        Rows(l, u, t=t).check()
        Rows(l, u, t=t, p=0.97).check()
        Rows(l, u, t=t, k=3000, p=0.5).check()


def test_rows_of_any_stride(gpu_ready):
    rng = np.random.default_rng(3)
    l = logits_of(rng, 5, 1003)
    r = Rows(l, rng.random(5), t=0.9, k=30, p=0.9)
    want = r.check()
    wide = torch.full((5, 2050), 50.0, device="cuda")
    for at in (0, 1, 3, 1047):
        view = wide[:, at:at + 1003]
        view.copy_(r.logits)
        assert (r.run(view) == want).all()
        view.fill_(50.0)


@pytest.mark.parametrize("rows,vocab", [(40, 9000), (64, 151936), (300, 8192), (2000, 700), (65536, 3)])
def test_many_rows(gpu_ready, rows, vocab):
    """Shapes of every division into chunks and units, requests of every kind."""
    rng = np.random.default_rng(rows)
    l = logits_of(rng, rows, vocab)
    r = Rows(l, rng.random(rows), t=rng.choice([0.0, 0.5, 1.0, 1.4], rows), k=rng.choice([0, 1, 50, 5000], rows),
             p=rng.choice([0.3, 0.9, 1.0], rows), low=rng.choice([0.0, 0.02], rows))
    got = r.run()
    for i in rng.choice(rows, min(rows, 60), replace=False):
        want = answers(l[i], r.u[i], *(x[i] for x in r.par))
        assert int(got[i]) in want, (i, int(got[i]), want)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.05, 0.3])
@pytest.mark.parametrize("vocab", [3000, 60000])
def test_cuts_among_many_near_logits(gpu_ready, vocab, spread):
    """More tokens in the bins in question than are listed or sorted at once."""
    rng = np.random.default_rng(vocab)
    l = (spread * rng.standard_normal((8, vocab))).astype(np.float32)
    u, p = rng.random(8), np.array([0.01, 0.1, 0.3, 0.5, 0.77, 0.9, 0.999, 1.0])
    k = np.array([0, 100, vocab // 3, 0, vocab - 7, 5000, 0, vocab // 2])
    Rows(l, u, p=p).check()
    Rows(l, u, t=0.3, k=k).check()
    Rows(l, u, t=2.0, k=k, p=p, low=0.9).check()


def test_large_vocabulary(gpu_ready):
    rng = np.random.default_rng(9)
    l = logits_of(rng, 2, 1 << 20)
    Rows(l, [0.3, 0.95], p=0.9).check()
    Rows(l, [0.3, 0.95]).check()


def test_captured_with_other_parameters_at_each_replay(gpu_ready):
    rng = np.random.default_rng(11)
    rows, vocab = 9, 20000
    logits = torch.empty(rows, vocab, device="cuda")
    u, t, p, low = (torch.empty(rows, device="cuda") for _ in range(4))
    k = torch.empty(rows, dtype=torch.int32, device="cuda")
    out = torch.empty(rows, dtype=torch.int32, device="cuda")
    ws = D.sample_workspace(rows, vocab)
    D.sample(logits.zero_(), u.zero_(), out, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        D.sample(logits, u, out, ws, temperature=t, top_k=k, top_p=p, min_p=low)
    for i in range(5):
        r = Rows(logits_of(rng, rows, vocab), rng.random(rows), t=rng.choice([0, 0.5, 1.0], rows),
                 k=rng.choice([0, 1, 40], rows), p=rng.choice([0.5, 0.9, 1.0], rows),
                 low=rng.choice([0.0, 0.1], rows))
        logits.copy_(r.logits)
        for x, y in zip((u, t, k, p, low), (r.u, *r.par)):
            x.copy_(torch.from_numpy(y))
        out.fill_(-9)
        graph.replay()
        torch.cuda.synchronize()
        assert (out.cpu().numpy() == r.check()).all()


def test_two_calls_at_once(gpu_ready):
    rng = np.random.default_rng(12)
    made = [Rows(logits_of(rng, 20, 30000), rng.random(20), t=0.8, k=40, p=p) for p in (0.95, 0.6)]
    want = [torch.from_numpy(r.check()).cuda() for r in made]
    calls = []
    for r in made:
        t, k, p, _ = (None if x is None else torch.from_numpy(x).cuda() for x in r.par)
        calls.append(dict(logits=r.logits, u=torch.from_numpy(r.u).cuda(), temperature=t, top_k=k, top_p=p,
                          out=torch.zeros(20, dtype=torch.int32, device="cuda"),
                          workspace=D.sample_workspace(20, 30000)))
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for c, s in zip(calls, streams):
            D.sample(**c, stream=s)
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert torch.equal(c["out"], w)


def test_distribution(gpu_ready):
    """Evenly spread random numbers take each token as often as it weighs."""
    n = 4096
    l = np.log(np.array([[1, 2, 3, 4, 6]], np.float32)).repeat(n, 0)
    got = Rows(l, (np.arange(n) + 0.5) / n).run()
    assert np.abs(np.bincount(got, minlength=5) / n - np.array([1, 2, 3, 4, 6]) / 16).max() <= 1 / n


def test_refusals(gpu_ready):
    l = torch.zeros(3, 100, device="cuda")
    u, out = torch.zeros(3, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    ws = D.sample_workspace(3, 100)
    good = dict(logits=l, u=u, out=out, workspace=ws)
    D.sample(**good)
    for bad in (dict(logits=l.double()), dict(logits=l[0]), dict(logits=l.t()), dict(logits=l.cpu()),
                dict(u=u[:2]), dict(u=u.double()), dict(u=u.cpu()), dict(out=out.long()), dict(out=out[:2]),
                dict(temperature=u[:1]), dict(top_k=u), dict(top_p=out), dict(min_p=u.half()),
                dict(workspace=ws.cpu())):
        with pytest.raises(ValueError):
            D.sample(**{**good, **bad})
    with pytest.raises(RuntimeError):
        D.sample_workspace(3, (1 << 20) + 1)
    with pytest.raises(RuntimeError):
        D.sample(l.expand(3, 100)[:1].expand(3, 100), u, out, ws)      # rows on top of each other
    with pytest.raises(RuntimeError):
        D.sample(l, u, out, ws[:-1])
    D.sample(torch.zeros(0, 100, device="cuda"), u[:0], out[:0], ws)
