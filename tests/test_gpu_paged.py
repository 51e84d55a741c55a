"""Keys and values in pages: dnx_paged_append and dnx_paged_attention against
the formulas in 64 bits.

Tolerances, with u = 2^-24. The append: a head's mean square is a sum of hd
squares in a tree of 8 or fewer additions (9 u), its root and inverse halve
that and add 3 u, two products add 2 u: a normed value is off by 10 u; the
rotation adds a rounding to each of its two products and one to their sum, so
|error| <= 13 u (|n1 c| + |n2 s|). In a bf16 cache half a step more: 2^-8 of
the value. Values that are only copied are equal to the bit.

The attention: a score is a sum of hd products on the matrix cores, off by
2 hd u sum|q k| / sqrt(hd) at most (2 u an addition: the unit's own rounding is
not documented); to that come the roundings of the score in units of log2 (2 u
|score|) and of exp2 (2 u). A weight's relative error e is the sum of these,
and the normalised weights are off by 2 e. The sums over N keys add 2 (N + 64)
u of the sum of |weight v|. So |error| <= (2 e + 2 (N + 64) u) sum_j p_j |v_j|
with e for the worst key of the row; the gate adds 4 u."""

import itertools

import numpy as np
import pytest
import torch

from dianoia_amd import device as D
from gpu_util import host

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-6


def rope_table(rows, hd):
    a = np.arange(rows)[:, None] / 10000.0 ** (np.arange(0, hd, 2) / hd)
    return np.concatenate([np.cos(a), np.sin(a)], 1).astype(np.float32)


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ the append

def rotated(x, norm, rope):
    """(value, sum of the sizes of its two terms) in 64 bits."""
    x = x.astype(np.float64)
    if norm is not None:
        r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(EPS)))
        x = norm.astype(np.float64) * x * r
    if rope is None:
        return x, np.abs(x)
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    c, s = (t[:, None].astype(np.float64) for t in (rope[:, :half], rope[:, half:]))
    return (np.concatenate([a * c - b * s, b * c + a * s], -1),
            np.concatenate([abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)], -1))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("n,heads,kv,hd,page,norm,rope,fused", [
    (1, 16, 8, 128, 16, True, True, True), (1, 1, 1, 64, 16, True, True, False),
    (5, 3, 1, 64, 32, True, True, True), (37, 12, 4, 128, 64, False, True, True),
    (130, 8, 8, 64, 16, True, False, True), (33, 0, 2, 128, 128, True, True, False),
    (64, 6, 2, 64, 256, False, False, False), (1000, 32, 8, 128, 64, True, True, True)])
def test_append(gpu_ready, kind, n, heads, kv, hd, page, norm, rope, fused):
    rng = np.random.default_rng(n + heads + hd)
    pages, rows = -(-n // page) + 3, 700
    dims = (heads + 2 * kv) * hd
    x = rng.standard_normal((n, dims)).astype(np.float32)
    xd = torch.from_numpy(x).cuda()
    parts = [xd[:, :heads * hd], xd[:, heads * hd:(heads + kv) * hd], xd[:, (heads + kv) * hd:]]
    if not fused:
        parts = [p.contiguous() for p in parts]
    q, k, v = (p.view(n, -1, hd) for p in parts)
    qh, kh, vh = (x[:, a:b].reshape(n, -1, hd) for a, b in
                  ((0, heads * hd), (heads * hd, (heads + kv) * hd), ((heads + kv) * hd, dims)))
    table = rope_table(rows, hd)
    pos = rng.integers(0, rows, n)
    slots = rng.permutation(pages * page)[:n]
    if n > 4:   # tokens that are left out: padding, past the cache, past the table
        slots[1], slots[2] = -1, pages * page
        if rope:
            pos[3], pos[4] = rows, -1
    live = (slots >= 0) & (slots < pages * page)
    if rope:
        live &= (pos >= 0) & (pos < rows)
    qw, kw = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    keys, values = (torch.randn(pages, page, kv, hd, device="cuda").to(TYPES[kind]) for _ in range(2))
    before = [t.clone() for t in (keys, values)]
    q_out = torch.full((n, max(heads, 1), hd), 9.0, device="cuda")
    dev = lambda t: torch.from_numpy(t).cuda()
    D.paged_append(D.PagedCache(keys, values), k, v, ints(pos), ints(slots),
                   rope=dev(table) if rope else None, q=q if heads else None,
                   q_out=q_out if heads else None, q_norm=dev(qw) if norm else None,
                   k_norm=dev(kw) if norm else None, eps=EPS)
    rows_of = table[np.clip(pos, 0, rows - 1)] if rope else None
    step = 0.0 if kind == "f32" else 2.0 ** -8
    if heads:
        want, size = rotated(qh, qw if norm else None, rows_of)
        got = host(q_out)
        assert (np.abs(got - want) <= 13 * U * size)[live].all()
        assert (got[~live] == 9.0).all()
    want, size = rotated(kh, kw if norm else None, rows_of)
    got = keys.view(-1, kv, hd).double().cpu().numpy()
    err = np.abs(got[slots[live]] - want[live])
    assert (err <= (13 * U * size + step * (np.abs(want) + 13 * U * size))[live]).all()
    flat = values.view(-1, kv, hd)
    at = ints(slots[live]).long()
    assert torch.equal(flat[at], dev(vh[live]).to(TYPES[kind]))
    untouched = np.ones(pages * page, bool)
    untouched[slots[live]] = False
    where = torch.from_numpy(untouched).cuda()
    for t, old in zip((keys, values), before):
        assert torch.equal(t.view(-1, kv, hd)[where], old.view(-1, kv, hd)[where])


def test_append_q_in_place(gpu_ready):
    n, heads, kv, hd = 19, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(n, h, hd, device="cuda", generator=g) for h in (heads, kv, kv))
    rope = torch.from_numpy(rope_table(64, hd)).cuda()
    w = torch.ones(hd, device="cuda")
    keys, values = torch.zeros(2, 16, kv, hd, device="cuda"), torch.zeros(2, 16, kv, hd, device="cuda")
    out = torch.empty_like(q)
    args = (D.PagedCache(keys, values), k, v, ints(range(n)), ints(range(n)))
    D.paged_append(*args, rope=rope, q=q, q_out=out, q_norm=w, k_norm=w)
    D.paged_append(*args, rope=rope, q=q, q_out=q, q_norm=w, k_norm=w)
    assert torch.equal(q, out)


def test_append_single_heads_of_any_stride(gpu_ready):
    """A dimension of one has no stride: a tensor [1][n][hd] turned to [n][1][hd]."""
    n, hd = 7, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(1, n, hd, device="cuda", generator=g) for _ in range(3))
    rope = torch.from_numpy(rope_table(64, hd)).cuda()
    got = []
    for turn in (lambda t: t.transpose(0, 1), lambda t: t.view(n, 1, hd)):
        keys, values = (torch.zeros(1, 16, 1, hd, device="cuda") for _ in range(2))
        q_out = torch.zeros(n, 1, hd, device="cuda")
        D.paged_append(D.PagedCache(keys, values), turn(k), turn(v), ints(range(n)), ints(range(n)),
                       rope=rope, q=turn(q), q_out=q_out)
        got.append((keys, values, q_out))
    for a, b in zip(*got):
        assert torch.equal(a, b) and bool(a.any())


# --------------------------------------------------------------- the attention

class Batch:
    """A batch whose cache holds NaN wherever no sequence's key lies."""

    def __init__(self, seed, counts, lens, prefix, heads, kv, hd, kind, page, pad=0, gate=False,
                 max_len=None, spare=2, scale=2.0):
        rng = np.random.default_rng(seed)
        self.counts, self.lens, self.prefix = list(counts), list(lens), prefix
        self.heads, self.kv, self.hd, self.page = heads, kv, hd, page
        need = [-(-n // page) for n in lens]
        shared = -(-prefix // page)
        pages = shared + sum(need) + spare
        order = rng.permutation(pages).astype(np.int32)
        self.keys, self.values = (torch.full((pages, page, kv, hd), float("nan"), device="cuda",
                                             dtype=TYPES[kind]) for _ in range(2))
        width = max(max(need), 1) + 1
        tables = np.full((len(lens), width), -7, np.int32)   # entries past a sequence's pages
        self.shared = order[:shared]
        at = shared
        for b, c in enumerate(need):
            tables[b, :c] = order[at:at + c]
            at += c
        self.tables_h = tables
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.own_kv, self.first_kv = [], None
        for pages_of, count, keep in [(self.shared, prefix, None)] + [
                (tables[b], n, b) for b, n in enumerate(lens)]:
            kvs = []
            for t in (self.keys, self.values):
                x = torch.randn(count, kv, hd, device="cuda", generator=g).to(t.dtype)
                for i in range(0, count, page):
                    t[int(pages_of[i // page]), :min(page, count - i)] = x[i:i + page]
                kvs.append(x)
            if keep is None:
                self.first_kv = kvs
            else:
                self.own_kv.append(kvs)
        self.live = sum(counts)
        rows = self.live + pad
        self.q = scale * torch.randn(rows, heads, hd, device="cuda", generator=g)
        if pad:
            self.q[self.live:] = float("nan")
        self.gate = torch.randn(rows, heads, device="cuda", generator=g) if gate else None
        self.cache = D.PagedCache(self.keys, self.values)
        self.starts = ints(np.concatenate([[0], np.cumsum(counts)]))
        self.lens_d, self.tables = ints(lens), ints(tables)
        self.max_len = max(lens) if max_len is None else max_len
        self.batch = D.PagedBatch(self.starts, self.lens_d, self.tables, rows, max(max(counts), 1),
                                  self.max_len, prefix_pages=ints(self.shared) if shared else None,
                                  prefix_len=prefix)
        self.out = torch.full((rows, heads, hd), 3.25, device="cuda")
        self.ws = D.paged_attention_workspace(self.cache, self.batch, heads)
        self.ws.fill_(0xff)   # NaN: what is read of it has been written

    def run(self, window=0, stream=None):
        D.paged_attention(self.cache, self.batch, self.q, self.out, self.ws, window=window,
                          gate=self.gate, stream=stream)
        return self.out

    def expected(self, window=0, seen=None):
        """(value, bound on the error) per row in 64 bits; seen(b, j): whether
        key j of sequence b (its prefix's keys first) exists."""
        want = np.zeros((self.live, self.heads, self.hd))
        room = np.zeros_like(want)
        group, t = self.heads // self.kv, 0
        q = self.q[:self.live].double().cpu().numpy()
        gate = None if self.gate is None else self.gate[:self.live].double().cpu().numpy()
        for b, (c, n) in enumerate(zip(self.counts, self.lens)):
            n_seen = min(n, self.max_len)
            k, v = (np.concatenate([f.double().cpu().numpy(), o.double().cpu().numpy()[:n_seen]])
                    for f, o in zip(self.first_kv, self.own_kv[b]))
            there = np.array([seen is None or seen(b, j) for j in range(len(k))], bool)
            for i in range(c):
                p = self.prefix + n - c + i
                j = np.arange(len(k))
                ok = there & (j <= p) & ((j > p - window) if window else True)
                if ok.any():
                    kk, vv = k[ok], v[ok]
                    for h in range(self.heads):
                        s = kk[:, h // group] @ q[t, h] / np.sqrt(self.hd)
                        size = np.abs(kk[:, h // group]) @ np.abs(q[t, h]) / np.sqrt(self.hd)
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        e = (2 * self.hd * U * size + 2 * U * np.abs(s)).max() + 2 * U
                        want[t, h] = w @ vv[:, h // group]
                        room[t, h] = (2 * e + 2 * (len(kk) + 64) * U) * (w @ np.abs(vv[:, h // group]))
                        if gate is not None:
                            g = 1 / (1 + np.exp(-gate[t, h]))
                            room[t, h] = (room[t, h] + 4 * U * np.abs(want[t, h])) * g
                            want[t, h] *= g
                t += 1
        return want, room

    def check(self, window=0, seen=None):
        out = host(self.run(window))
        want, room = self.expected(window, seen)
        err = np.abs(out[:self.live] - want)
        assert np.isfinite(out[:self.live]).all()
        assert (err <= room + 1e-37).all(), (float((err / (room + 1e-37)).max()), float(err.max()))
        assert (out[self.live:] == 3.25).all()
        return out


CASES = [
    # counts, lens, prefix, heads, kv, hd, page
    ([1], [1], 0, 1, 1, 64, 16),
    ([1], [17], 0, 16, 8, 128, 16),
    ([1, 1, 1], [33, 200, 64], 0, 8, 2, 64, 16),
    ([1] * 5, [1, 16, 31, 32, 100], 100, 8, 8, 128, 32),
    ([1] * 9, [5, 60, 61, 700, 12, 300, 1, 2, 3], 257, 12, 4, 64, 64),
    ([2, 0, 5, 1, 0], [2, 30, 90, 400, 0], 65, 6, 2, 128, 16),
    ([37, 1, 12], [37, 500, 100], 777, 12, 4, 64, 16),
    ([70], [130], 0, 5, 1, 64, 32),
    ([1, 1], [300, 2], 1, 33, 1, 64, 16),
    ([3, 3], [3, 3], 4100, 8, 2, 128, 256),
    ([1] * 40, list(range(1, 41)), 520, 16, 2, 128, 16),
    ([1, 1], [3000, 1500], 0, 4, 4, 128, 128),
    ([1] * 40, [30] * 40, 1500, 16, 2, 128, 64),
    ([200, 1, 90], [333, 70, 90], 190, 4, 2, 64, 32),
    ([150], [700], 64, 3, 1, 128, 16),
]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention(gpu_ready, case, kind):
    counts, lens, prefix, heads, kv, hd, page = CASES[case]
    Batch(case, counts, lens, prefix, heads, kv, hd, kind, page, pad=case % 3,
          gate=case % 2 == 1).check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 16, 50, 130, 512, 100000])
def test_window(gpu_ready, window, kind):
    """Windows that end in the prefix, in the own keys, and before both."""
    for counts, lens, prefix in (([1] * 4, [1, 40, 90, 600], 200), ([9, 30, 1], [9, 64, 300], 70),
                                 ([20], [150], 0)):
        Batch(window, counts, lens, prefix, 6, 2, 64, kind, 16, pad=1).check(window)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 70, 700])
def test_many_sequences_of_unequal_lengths(gpu_ready, window, kind):
    """Sequences without tokens, without keys, of one key, of whole steps, and one
    that is most of the batch; a bound on the lengths that is far above them."""
    rng = np.random.default_rng(17)
    lens = rng.choice([0, 1, 5, 63, 64, 65, 128, 200, 333, 900], 130).tolist()
    counts = [min(int(c), max(n, 1)) for c, n in zip(rng.choice([0, 1, 1, 1, 2, 8], 130), lens)]
    Batch(20, counts, lens, 100, 4, 2, 64, kind, 16, pad=3, gate=True).check(window)
    one = [0] * 40 + [1] + [0] * 88 + [1]
    Batch(21, one, [2000 if c else 0 for c in one], 0, 4, 2, 128, kind, 64).check(window)
    Batch(22, [1] * 64, list(range(64)), 0, 8, 4, 64, kind, 16, max_len=100000).check(window)
    for seqs in (256, 257):
        lens = [int(n) for n in rng.integers(0, 40, seqs)]
        lens[3] = lens[-1] = 600
        Batch(seqs, [1] * seqs, lens, 65, 2, 1, 64, kind, 32).check(window)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_without_keys_are_zeros(gpu_ready, kind):
    """A token that stands before its sequence's first own key, and no prefix."""
    b = Batch(3, [1, 2, 1], [0, 1, 20], 0, 4, 2, 64, kind, 16, pad=2)
    out = b.check()
    assert (out[0] == 0).all() and (out[1] == 0).all() and (out[2] != 0).any()
    b = Batch(3, [1], [0], 0, 4, 2, 64, kind, 16)      # no key in the whole call
    assert (b.check() == 0).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [1, 16, 63, 64, 65, 128, 250])
def test_short_prefix(gpu_ready, prefix, kind):
    """A prefix and own keys that one workgroup walks, with own keys that begin
    at a step's start and windows that end anywhere; sequences without tokens
    and tables with pages outside the cache."""
    for (heads, kv, hd, page), counts in itertools.product(
            [(2, 2, 64, 16), (6, 2, 128, 64), (8, 1, 64, 32)], [[1, 1, 0, 1], [3, 1, 2, 0]]):
        b = Batch(prefix, counts, [60, 1, 33, 4], prefix, heads, kv, hd, kind, page, pad=1, gate=True)
        for window in (0, 1, 5, 40, 64, prefix, prefix + 1, 100, 1000):
            b.check(window)
        b.batch.prefix_pages[-1] = -1
        b.tables[0, 0] = 0x7fffffff
        last = (prefix - 1) // page * page
        b.check(seen=lambda s, j: j < last if j < prefix else s != 0 or j - prefix >= page)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("counts,lens,prefix,heads,hd", [
    ([1], [70001], 0, 2, 64), ([2, 1], [33000, 5], 40000, 3, 64), ([1], [20], 66000, 9, 128)])
def test_many_runs(gpu_ready, counts, lens, prefix, heads, hd, kind):
    """Long caches of one key head: up to 256 runs to add, most of them empty
    under a window."""
    b = Batch(13, counts, lens, prefix, heads, 1, hd, kind, 256, pad=1, gate=True)
    b.check()
    b.check(3000)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_short_prefix_and_no_own_key(gpu_ready, kind):
    b = Batch(10, [1, 1], [0, 2], 20, 4, 2, 64, kind, 16)
    out = host(b.run())
    alone = Batch(10, [1, 1], [0, 0], 20, 4, 2, 64, kind, 16)
    alone.q.copy_(b.q)
    for t in ("keys", "values"):
        getattr(alone, t)[torch.from_numpy(alone.shared).cuda().long()] = \
            getattr(b, t)[torch.from_numpy(b.shared).cuda().long()]
    alone.first_kv = b.first_kv
    want, room = alone.expected()       # places 19: all twenty keys
    assert (np.abs(out[0] - want[0]) <= room[0]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_page_listed_more_than_once(gpu_ready, kind):
    """By two sequences, twice by one, and among the prefix's pages."""
    b = Batch(11, [1, 2, 1], [70, 64, 33], 300, 8, 4, 64, kind, 32)
    b.tables[0, 1] = b.tables[0, 0]
    b.tables[1, 0] = b.tables[2, 0]
    b.batch.prefix_pages[3] = b.tables[2, 0]
    for x, own in zip(b.first_kv, zip(*b.own_kv)):
        own[0][32:64] = own[0][:32]
        own[1][:32] = own[2][:32]
        x[96:128] = own[2][:32]
    b.check()
    b.check(40)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_two_calls_at_once(gpu_ready, kind):
    """On two streams, with a workspace each, over one cache."""
    a = Batch(12, [1] * 9, [40 * i + 1 for i in range(9)], 700, 8, 4, 64, kind, 32)
    b = Batch(12, [1] * 9, [40 * i + 1 for i in range(9)], 700, 8, 4, 64, kind, 32)
    b.q.mul_(0.5)
    b.cache = a.cache
    want = host(a.run()), host(b.run())
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for x, s in zip((a, b), streams):
        x.out.zero_()
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for x, s in zip((a, b), streams):
            x.run(stream=s)
    torch.cuda.synchronize()
    for x, w in zip((a, b), want):
        assert np.array_equal(host(x.out), w)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_more_tokens_than_own_keys(gpu_ready, kind):
    """The first of them see the prefix alone, under the widest window too."""
    b = Batch(9, [3], [1], 50, 4, 2, 64, kind, 16)
    want, room = b.expected()                      # of the last, which sees all 51 keys
    longer = Batch(9, [1], [0], 50, 4, 2, 64, kind, 16)
    for window in (0, 0x7fffffff):
        out = host(b.run(window))
        assert (np.abs(out[2] - want[2]) <= room[2]).all()
        for i in (0, 1):
            longer.q.copy_(b.q[i:i + 1])
            longer.first_kv = b.first_kv
            got, bound = longer.expected()
            assert (np.abs(out[i] - got[0]) <= bound[0]).all(), (window, i)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 5000, 0x7ffffffd, 0x7fffffff])
@pytest.mark.parametrize("count,own,other,prefix,heads", [
    (8, 4, 2000, 0, 4), (70, 66, 2000, 0, 4), (6, 2, 1, 500, 4), (6, 0, 900, 500, 2), (100, 3, 300, 500, 6)])
def test_tokens_before_their_own_keys_in_many_runs(gpu_ready, count, own, other, prefix, heads, window,
                                                   kind):
    """More new tokens than own keys in calls that add partial results, under
    windows whose first key lies 2^31 places before the token: the first tokens
    see the prefix alone (or nothing), the last ones all up to their own key."""
    b = Batch(count, [count, 1], [own, other], prefix, heads, 2, 64, kind, 16)
    assert b.ws.numel() > 4 * heads * 64          # partial results
    out = host(b.run(window))
    want, room = b.expected()                     # the rows whose place is a key's
    rest = count - own
    assert (np.abs(out[rest:] - want[rest:]) <= room[rest:]).all()
    if prefix == 0:
        assert (out[:rest] == 0).all()
        return
    for i in range(0, rest, 7):                   # a token at the prefix's last key sees all of it
        alone = Batch(count, [1], [0], prefix, heads, 2, 64, kind, 16)
        alone.first_kv = b.first_kv
        alone.q.copy_(b.q[i:i + 1])
        want, room = alone.expected()
        assert (np.abs(out[i] - want[0]) <= room[0]).all(), i


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [40, 500])
@pytest.mark.parametrize("counts", [[1, 1], [1, 5], [70, 2]])
def test_a_window_far_behind_the_keys(gpu_ready, counts, prefix, kind):
    """Lengths past the bound, up to the largest: such a token stands behind
    every key, and under a window sees none of them."""
    b = Batch(15, counts, [60, 20], prefix, 4, 2, 64, kind, 16)
    for far in (1 << 20, 0x7fffffff - prefix, 0x7fffffff):
        b.lens_d.fill_(far)
        for window in (1, 50, 100000):
            assert (host(b.run(window)) == 0).all(), (far, window)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,seqs,tokens,most,page,width,prefix", [
    (8, 8, 4096, 4200, 4200, 64, 290, 0), (8, 8, 4096, 4200, 4200, 64, 290, 300),
    (16, 16, 65536, 2000, 20, 256, 71, 0), (4, 1, 50000, 4200, 4200, 256, 70, 40)])
def test_bounds_far_above_the_batch(gpu_ready, heads, kv, seqs, tokens, most, page, width, prefix, kind):
    """Many sequences that might each have many tokens and a long cache, of
    which a few have any: the bounds' product is more workgroups than a launch
    may have."""
    counts, lens = [19, 1, 7, 2, 20], [40, 600, 7, 1, 333]
    if most > 100:
        counts[0], lens[0] = 150, 180
    b = Batch(17, counts, lens, prefix, heads, kv, 64, kind, page, pad=5, gate=True)
    rng = np.random.default_rng(seqs)
    at = np.sort(rng.permutation(np.arange(1, seqs - 1))[:3])
    at = np.concatenate([[0], at, [seqs - 1]])    # the first and the last among them
    n, own = np.zeros(seqs, np.int64), np.zeros(seqs, np.int64)
    n[at], own[at] = counts, lens
    tables = np.full((seqs, width), -7, np.int32)
    tables[at, :b.tables_h.shape[1]] = b.tables_h
    rows = b.live + 5
    q = torch.full((tokens, heads, 64), float("nan"), device="cuda")
    q[:rows], gate = b.q, torch.zeros(tokens, heads, device="cuda")
    gate[:rows] = b.gate
    b.q, b.gate = q, gate
    b.out = torch.full((tokens, heads, 64), 3.25, device="cuda")
    b.batch = D.PagedBatch(ints(np.concatenate([[0], np.cumsum(n)])), ints(own), ints(tables), tokens,
                           most, width * page, prefix_pages=b.batch.prefix_pages if prefix else None,
                           prefix_len=prefix)
    b.ws = D.paged_attention_workspace(b.cache, b.batch, heads)
    b.ws.fill_(0xff)
    b.check()
    b.check(100)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 90])
def test_a_prompt_among_single_tokens(gpu_ready, window, kind):
    """One long prompt beside decoding sequences, and others without a token or
    of a few: most sequences have few of the blocks that the longest has. And
    prompts alone, on few key heads."""
    counts = [1] * 40 + [210] + [1, 0, 3, 17] * 8
    lens = [max(c, 5 * i + 1) for i, c in enumerate(counts)]
    Batch(31, counts, lens, 0, 8, 4, 64, kind, 16, pad=2, gate=True).check(window)
    Batch(32, counts, lens, 300, 4, 4, 64, kind, 32, pad=70).check(window)
    short = [min(c, 17) for c in counts]
    Batch(33, short, lens, 0, 64, 32, 64, kind, 64).check(window)
    Batch(34, [900, 300], [900, 400], 0, 6, 1, 64, kind, 64, pad=1).check(window)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 32, 500])
def test_lengths_past_the_bound(gpu_ready, prefix, kind):
    """lens far past max_len: the keys up to max_len count, those in listed
    pages of the cache, and a table's other entries none."""
    b = Batch(18, [1, 2], [100, 48], prefix, 4, 2, 64, kind, 16)   # 7 and 3 pages; the others -7
    b.lens = [1 << 30, 1 << 30]
    b.lens_d.copy_(ints(b.lens))
    out = b.check().copy()
    b.lens_d.copy_(ints([100, 1000]))
    assert np.array_equal(out, host(b.run()))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 200])
def test_another_prompt_at_each_replay(gpu_ready, prefix, kind):
    """One captured call whose rows are another sequence's at each replay: the
    prompt of 150 tokens moves, the others have one token or none."""
    seqs, heads, kv, lens = 48, 8, 8, [200 + i for i in range(48)]
    ones = Batch(41, [1] * seqs, lens, prefix, heads, kv, 64, kind, 32, gate=True)
    rows = 150 + seqs
    g = torch.Generator(device="cuda").manual_seed(6)
    ones.q = 2 * torch.randn(rows, heads, 64, device="cuda", generator=g)
    ones.gate = torch.randn(rows, heads, device="cuda", generator=g)
    ones.out = torch.full((rows, heads, 64), 3.25, device="cuda")
    ones.batch = D.PagedBatch(ones.starts, ones.lens_d, ones.tables, rows, 150, max(lens),
                              prefix_pages=ones.batch.prefix_pages, prefix_len=prefix)
    ones.ws = D.paged_attention_workspace(ones.cache, ones.batch, heads)
    ones.ws.fill_(0xff)
    ones.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ones.run()
    for at in (0, 17, seqs - 1, 5):
        counts = [1 if (i + at) % 3 else 0 for i in range(seqs)]
        counts[at] = 150
        ones.counts, ones.live = counts, sum(counts)
        ones.starts.copy_(ints(np.concatenate([[0], np.cumsum(counts)])))
        ones.out.fill_(3.25)
        graph.replay()
        torch.cuda.synchronize()
        got = ones.out.clone()
        ones.out.fill_(3.25)
        ones.check()
        assert torch.equal(got, ones.out)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_pages_outside_the_cache_are_not_seen(gpu_ready, kind):
    b = Batch(4, [1, 3], [100, 90], 64, 8, 4, 128, kind, 16)
    b.tables[0, 2], b.tables[1, 0] = -1, b.keys.shape[0]
    b.tables[1, 3] = 0x7fffffff
    missing = {0: [2], 1: [0, 3]}
    b.check(seen=lambda s, j: j < 64 or (j - 64) // 16 not in missing[s])
    b.tables.fill_(-1)
    b.check(seen=lambda s, j: j < 64)
    b = Batch(5, [2], [40], 0, 2, 2, 64, kind, 32)
    b.tables.fill_(1 << 30)
    assert (host(b.run()) == 0).all()


def test_keys_past_the_bounds_are_not_seen(gpu_ready):
    """lens past max_len, and past the pages of the table."""
    b = Batch(6, [1, 1], [100, 40], 32, 4, 2, 64, "f32", 16, max_len=48)
    b.check()
    b = Batch(7, [1, 1], [100, 40], 32, 4, 2, 64, "f32", 16)
    b.lens_d.fill_(1 << 30)       # tables of 8 pages, of which 7 and 3 are listed
    b.max_len = 100
    out = host(b.run())
    b.lens = [100, 48]
    b.lens_d.copy_(ints([100, 48]))
    assert np.isfinite(out[0]).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 32, 500])
def test_keys_past_the_table_are_not_seen(gpu_ready, prefix, kind):
    """A length, and a bound on it, past the pages that a table lists."""
    b = Batch(16, [1, 1], [48, 48], prefix, 4, 2, 64, kind, 16)
    tables = b.tables[:, :3].contiguous()
    b.batch = D.PagedBatch(b.starts, b.lens_d, tables, 2, 1, 1 << 20,
                           prefix_pages=b.batch.prefix_pages, prefix_len=prefix)
    b.ws = D.paged_attention_workspace(b.cache, b.batch, 4)
    b.ws.fill_(0xff)
    b.lens_d.copy_(ints([1 << 20, 60]))
    b.check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("heads,kv,hd,page", [(4, 2, 64, 16), (64, 2, 64, 64), (64, 1, 128, 16),
                                              (64, 1, 128, 128)])
def test_infinities_behind_the_mask(gpu_ready, heads, kv, hd, page, kind):
    """An infinity or NaN among the keys or values of a later token does not
    reach the earlier ones; where it is seen, it follows the formula. The rows
    next to it may be formed by other instructions (float32 products in place
    of pieces), each within the bound of the formula on the clean cache."""
    counts, lens, prefix = [6], [40], 50
    make = lambda: Batch(8, counts, lens, prefix, heads, kv, hd, kind, page)
    want, room = make().expected()
    near = lambda got, at: (np.abs(got - want[at]) <= room[at]).all()
    for what in ("keys", "values"):
        for bad in (np.inf, -np.inf, np.nan):
            b = make()
            j = 37                                  # seen by tokens 3, 4 and 5 (places 37 .. 39)
            getattr(b, what)[int(b.tables_h[0, j // page]), j % page, :, 5] = bad
            out = host(b.run())
            assert near(out[:3], np.s_[:3]), (what, bad)
            if what == "values":
                assert near(out[3:, :, :5], np.s_[3:, :, :5])
                got = out[3:, :, 5]
                assert (np.isnan(got) if np.isnan(bad) else got == bad).all()
    b = make()                                  # a window hides the prefix's first keys
    want, room = b.expected(60)
    for t in (b.keys, b.values):
        t[int(b.shared[0]), :2] = float("nan")
    assert near(host(b.run(60)), np.s_[:])


def test_scores_that_overflow(gpu_ready):
    """-inf scores have no weight; a row of nothing else is zeros; +inf is NaN."""
    b = Batch(9, [1, 1], [20, 20], 0, 1, 1, 64, "f32", 32)
    b.q.zero_()
    b.q[:, 0, 0] = 1.0
    for s in range(2):
        page = int(b.tables_h[s, 0])
        b.keys[page, :20] = 0.0
        b.keys[page, :10, 0, 0] = -float("inf")
    b.keys[int(b.tables_h[1, 0]), 3, 0, 0] = float("inf")
    out = host(b.run())
    v = b.own_kv[0][1].double().cpu().numpy()[10:, 0].mean(0)
    assert np.abs(out[0, 0] - v).max() < 1e-6 and np.isnan(out[1]).all()
    for s in range(2):
        b.keys[int(b.tables_h[s, 0]), :20, 0, 0] = -float("inf")
    assert (host(b.run()) == 0).all()


def test_large_scores(gpu_ready):
    """Scores of thousands: one key takes the weight, nothing overflows."""
    Batch(10, [1, 4], [70, 80], 130, 8, 2, 128, "f32", 16, scale=300.0).check()


def test_offsets_past_32_bits(gpu_ready):
    """A cache of more than 2^32 bytes and 2^31 values, its last pages used."""
    pages, page, kv, hd = 66000, 32, 8, 128     # 2.16e9 values each
    keys, values = (torch.empty(pages, page, kv, hd, device="cuda") for _ in range(2))
    small = Batch(11, [1, 2], [50, 70], 40, 8, 8, 128, "f32", 32)
    want = host(small.run()).copy()
    shift = pages - small.keys.shape[0]
    keys[shift:], values[shift:] = small.keys, small.values
    cache = D.PagedCache(keys, values)
    batch = D.PagedBatch(small.starts, small.lens_d, small.tables + shift, 3, 2, 70,
                         prefix_pages=ints(small.shared + shift), prefix_len=40)
    out = torch.empty_like(small.out)
    D.paged_attention(cache, batch, small.q, out, small.ws)
    assert np.array_equal(host(out), want)
    k = torch.randn(1, kv, hd, device="cuda")
    D.paged_append(cache, k, k, None, ints([pages * page - 1]))
    assert torch.equal(keys[-1, -1], k[0]) and torch.equal(values[-1, -1], k[0])


def test_most_rows(gpu_ready):
    """As many rows as a call may have, nearly all of them padding."""
    rows, heads, kv = 1082401, 62, 31             # 2^26 - 2 rows of the result
    b = Batch(14, [3], [40], 500, heads, kv, 64, "bf16", 16)
    batch = D.PagedBatch(b.starts, b.lens_d, b.tables, rows, 3, 40,
                         prefix_pages=b.batch.prefix_pages, prefix_len=500)
    ws = D.paged_attention_workspace(b.cache, batch, heads)
    assert ws.numel() > 0
    q, out = (torch.empty(rows, heads, 64, device="cuda") for _ in range(2))
    q[:3] = b.q
    out.fill_(3.25)
    D.paged_attention(b.cache, batch, q, out, ws)
    want, room = b.expected()
    assert (np.abs(host(out[:3]) - want) <= room).all()
    assert not bool((out[3:] != 3.25).any())


def test_same_bits_again_on_another_stream(gpu_ready):
    b = Batch(12, [1] * 20, list(range(30, 230, 10)), 1000, 16, 4, 128, "f32", 32)
    first = b.run().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b.out.fill_(0)
    side.wait_stream(torch.cuda.current_stream())
    b.run(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(b.out, first)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_steps_together_eager_and_captured(gpu_ready, kind):
    """Decode steps as a server runs them: append, then attention, over growing
    sequences, once eagerly and once as one captured graph whose arrays change,
    with the program's own work between the replays. Every step against the
    formula on what the cache should hold."""
    seqs, prefix, heads, kv, hd, page, steps = 5, 75, 8, 2, 64, 16, 6
    pad = 3
    rng = np.random.default_rng(13)
    g = torch.Generator(device="cuda").manual_seed(13)
    width = 6
    pages = 8 + seqs * width
    order = rng.permutation(pages).astype(np.int32)
    shared, tables_h = order[:5], order[5:5 + seqs * width].reshape(seqs, width)
    rope = torch.from_numpy(rope_table(512, hd)).cuda()
    w = 1 + 0.1 * torch.randn(hd, device="cuda", generator=g)
    rows = seqs + pad
    step_qkv = [torch.randn(rows, (heads + 2 * kv) * hd, device="cuda", generator=g)
                for _ in range(steps)]
    begin = [3, 17, 40, 15, 60]
    history = [torch.randn(n, 2 * kv * hd, device="cuda", generator=g) for n in [prefix] + begin]

    def play(captured):
        keys, values = (torch.full((pages, page, kv, hd), float("nan"), device="cuda",
                                   dtype=TYPES[kind]) for _ in range(2))
        cache = D.PagedCache(keys, values)
        for i, x in enumerate(history):     # prompts, appended many tokens at once
            n = x.shape[0]
            table = shared if i == 0 else tables_h[i - 1]
            own = np.arange(n)
            D.paged_append(cache, x[:, :kv * hd].view(n, kv, hd), x[:, kv * hd:].view(n, kv, hd),
                           ints(own + (0 if i == 0 else prefix)),
                           ints(table[own // page] * page + own % page), rope=rope, k_norm=w)
        starts = ints(list(range(seqs + 1)))
        lens, tables = ints(begin), ints(tables_h)
        positions, slots = ints([0] * rows), ints([-1] * rows)
        qkv = torch.empty(rows, (heads + 2 * kv) * hd, device="cuda")
        q = qkv[:, :heads * hd].view(rows, heads, hd)
        k = qkv[:, heads * hd:(heads + kv) * hd].view(rows, kv, hd)
        v = qkv[:, (heads + kv) * hd:].view(rows, kv, hd)
        q_rot = torch.zeros(rows, heads, hd, device="cuda")
        out = torch.zeros(rows, heads, hd, device="cuda")
        batch = D.PagedBatch(starts, lens, tables, rows, 1, width * page, prefix_pages=ints(shared),
                             prefix_len=prefix)
        ws = D.paged_attention_workspace(cache, batch, heads)

        def step():
            D.paged_append(cache, k, v, positions, slots, rope=rope, q=q, q_out=q_rot, q_norm=w,
                           k_norm=w)
            D.paged_attention(cache, batch, q_rot, out, ws)

        graph = None
        got = []
        for i in range(steps):
            at = np.array(begin) + i
            lens.copy_(ints(at + 1))
            positions[:seqs] = ints(prefix + at)
            slots[:seqs] = ints(tables_h[np.arange(seqs), at // page] * page + at % page)
            qkv.copy_(step_qkv[i])
            if captured:
                if graph is None:           # capture runs nothing
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        step()
                graph.replay()
            else:
                step()
            got.append(out.clone())
            torch.cuda.synchronize()
        return keys, values, got

    keys, values, eager = play(False)
    keys2, values2, replayed = play(True)
    for a, b in zip(eager, replayed):
        assert torch.equal(a, b)
    same = lambda a, b: torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    assert same(keys, keys2) and same(values, values2)
    # The last step against the formula on the cache's own keys and values.
    i = steps - 1
    q, _ = rotated(step_qkv[i][:seqs, :heads * hd].cpu().numpy().reshape(seqs, heads, hd),
                   w.cpu().numpy(), rope.cpu().numpy()[prefix + np.array(begin) + i])
    flat = [t.view(-1, kv, hd).double().cpu().numpy() for t in (keys, values)]
    for b in range(seqs):
        n = begin[b] + steps
        places = np.concatenate([shared[np.arange(prefix) // page] * page + np.arange(prefix) % page,
                                 tables_h[b][np.arange(n) // page] * page + np.arange(n) % page])
        kk, vv = flat[0][places], flat[1][places]
        assert np.isfinite(kk).all() and np.isfinite(vv).all()
        for h in range(heads):
            s = kk[:, h // 4] @ q[b, h] / np.sqrt(hd)
            size = np.abs(kk[:, h // 4]) @ np.abs(q[b, h]) / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            # q itself is off by 13 u of its two terms (at most 1.5 times it)
            e = ((2 * hd + 20) * U * size + 2 * U * np.abs(s)).max() + 2 * U
            room = (2 * e + 2 * (len(kk) + 64) * U) * (p @ np.abs(vv[:, h // 4]))
            assert (np.abs(eager[i][b, h].double().cpu().numpy() - p @ vv[:, h // 4]) <= room).all()
    assert (eager[i][seqs:] == 0).all()
