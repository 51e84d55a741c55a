"""Keys and values in pages of int8 codes: dnx_paged_append, dnx_paged_read and
dnx_paged_attention on such a cache against the formulas in 64 bits.

Tolerances, with u = 2^-24. The append works in 64 bits: a code is that of the
formula unless 127 y / top lies within 1e-9 of the border of two codes, the
scale that of the formula rounded once (u, and 1e-15 of the doubles). Reading
back rounds one product: equal to code * scale in float32, to the bit.

The attention: a query is a multiple of 2^-22 of the power of two above its
largest value, off by 2^-22 of that value at most; its products with codes are
exact whole numbers, made floats by two roundings and scaled by four more, so a
score is off by 2^-22 max|q| sum|k| / sqrt(hd) + 8 u |s|; exp2 adds 2 u. A weight
times its value's scale is a multiple of 2^-22 of the power of two above the
largest of its step, off by 2^-22 of that one at most; steps are runs of up to
128 keys, so the largest lies within 127 keys of it. The sums over N keys add 2
(N + 64) u of the sum of |weight v| as on other caches, the gate 4 u."""

import itertools

import numpy as np
import pytest
import torch
from scipy.ndimage import maximum_filter1d

from dianoia_amd import device as D
from gpu_util import host
from test_gpu_sample import answers
from test_gpu_paged import CASES, EPS, U, Batch, ints, rope_table, rotated

pytestmark = pytest.mark.gpu


def empty_cache(pages, page, kv, hd):
    """Codes and scales whose unwritten places read as NaN."""
    codes = [torch.full((pages, page, kv, hd), 77, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.full((pages, kv, page), float("nan"), device="cuda") for _ in range(2)]
    return codes + scales


def stored(codes, scales):
    """[pages * page][kv_heads][hd] in 64 bits."""
    x = codes.double().cpu().numpy() * scales.double().cpu().numpy().transpose(0, 2, 1)[..., None]
    return x.reshape(-1, *x.shape[2:])


# ------------------------------------------------------------------ the append

def check_codes(codes, scales, want):
    """Codes and scales [n][kv_heads] against values in 64 bits."""
    top = np.abs(want).max(-1, keepdims=True)
    exact = 127 * want / np.where(top > 0, top, 1)
    code = np.sign(exact) * np.floor(np.abs(exact) + 0.5)
    sure = np.abs(np.abs(exact) % 1 - 0.5) > 1e-9
    assert (codes == code)[sure].all() and (np.abs(codes - exact) <= 0.5 + 1e-9).all()
    assert (np.abs(scales - top[..., 0] / 127) <= (U + 1e-14) * top[..., 0] / 127 + 2.0 ** -150).all()


@pytest.mark.parametrize("n,heads,kv,hd,page,norm,rope,fused", [
    (1, 16, 8, 128, 16, True, True, True), (1, 1, 1, 64, 16, True, True, False),
    (5, 3, 1, 64, 32, True, True, True), (37, 12, 4, 128, 64, False, True, True),
    (130, 8, 8, 64, 16, True, False, True), (33, 0, 2, 128, 128, True, True, False),
    (64, 6, 2, 64, 256, False, False, False), (1000, 32, 8, 128, 64, True, True, True)])
def test_append(gpu_ready, n, heads, kv, hd, page, norm, rope, fused):
    rng = np.random.default_rng(n + heads + hd)
    pages, rows = -(-n // page) + 3, 700
    dims = (heads + 2 * kv) * hd
    x = (rng.standard_normal((n, dims)) * np.exp(2 * rng.standard_normal((n, 1)))).astype(np.float32)
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
    cache = empty_cache(pages, page, kv, hd)
    q_out = torch.full((n, max(heads, 1), hd), 9.0, device="cuda")
    dev = lambda t: torch.from_numpy(t).cuda()
    D.paged_append(D.PagedCache(*cache), k, v, ints(pos), ints(slots),
                   rope=dev(table) if rope else None, q=q if heads else None,
                   q_out=q_out if heads else None, q_norm=dev(qw) if norm else None,
                   k_norm=dev(kw) if norm else None, eps=EPS)
    rows_of = table[np.clip(pos, 0, rows - 1)] if rope else None
    if heads:
        want, size = rotated(qh, qw if norm else None, rows_of)
        got = host(q_out)
        assert (np.abs(got - want) <= 13 * U * size)[live].all()
        assert (got[~live] == 9.0).all()
    untouched = np.ones(pages * page, bool)
    untouched[slots[live]] = False
    for i, want in ((0, rotated(kh, kw if norm else None, rows_of)[0]), (1, vh.astype(np.float64))):
        codes = host(cache[i]).reshape(-1, kv, hd)
        scales = host(cache[2 + i]).transpose(0, 2, 1).reshape(-1, kv)
        check_codes(codes[slots[live]].astype(np.float64), scales[slots[live]], want[live])
        assert (codes[untouched] == 77).all() and np.isnan(scales[untouched]).all()


@pytest.mark.parametrize("hd", [64, 128])
def test_append_special_values(gpu_ready, hd):
    """Zeros, an infinity, NaN, the smallest and the largest floats, values on
    the border of two codes."""
    n, kv = 7, 2
    x = np.random.default_rng(hd).standard_normal((n, kv, hd)).astype(np.float32)
    x[0] = 0
    x[1, 0, 3], x[1, 1, hd - 1] = np.inf, np.nan
    x[2] *= np.float32(1e-44)
    x[3, 0] = np.float32(3.0e38) * np.sign(x[3, 0])
    x[4, 0, :4] = [254, 1, 3, -5]           # 127 x / 254: halves, away from zero
    x[4, 0, 4:] = 0
    x[5, 1, :] = np.float32(-2.5)
    cache = empty_cache(1, 16, kv, hd)
    xd = torch.from_numpy(x).cuda()
    D.paged_append(D.PagedCache(*cache), xd, xd, None, ints(range(n)))
    for i in (0, 1):
        codes = host(cache[i])[0, :n].astype(np.float64)
        scales = host(cache[2 + i])[0].T[:n]
        assert np.isnan(scales[1]).all() and (codes[1] == 0).all()
        assert (scales[0] == 0).all() and (codes[0] == 0).all()
        assert codes[4, 0, :4].tolist() == [127, 1, 2, -3]
        assert (codes[5, 1] == -127).all()
        good = [2, 3, 4, 5, 6]
        check_codes(codes[good], scales[good], x[good].astype(np.float64))
    k = torch.full((1, kv, hd), 3e38, device="cuda")
    D.paged_append(D.PagedCache(*cache), k, k, None, ints([9]),
                   k_norm=torch.full((hd,), 3e38, device="cuda"))
    assert torch.isfinite(cache[2][0, :, 9]).all()     # the norm brings 3e38 to one
    rope = torch.full((1, hd), 3e38, device="cuda")
    D.paged_append(D.PagedCache(*cache), k, k, ints([0]), ints([10]), rope=rope)
    assert torch.isnan(cache[2][0, :, 10]).all() and (cache[0][0, 10] == 0).all()


# -------------------------------------------------------------------- the read

@pytest.mark.parametrize("kind", ["f32", "bf16", "i8"])
@pytest.mark.parametrize("n,kv,hd,page", [(1, 1, 64, 16), (1, 8, 128, 16), (37, 2, 64, 32),
                                          (300, 3, 128, 64), (1001, 8, 64, 128)])
def test_read(gpu_ready, n, kv, hd, page, kind):
    """Any places in any order, the same one twice, and rows that are left."""
    g = torch.Generator(device="cuda").manual_seed(n + hd)
    pages = 9
    x = [torch.randn(pages, page, kv, hd, device="cuda", generator=g) for _ in range(2)]
    if kind == "i8":
        codes = [(40 * t).round().clamp(-127, 127).to(torch.int8) for t in x]
        scales = [torch.rand(pages, kv, page, device="cuda", generator=g) for _ in range(2)]
        cache = D.PagedCache(*codes, *scales)
        values = [c.float() * s.transpose(1, 2)[..., None] for c, s in zip(codes, scales)]
    else:
        x = [t.to({"f32": torch.float32, "bf16": torch.bfloat16}[kind]) for t in x]
        cache = D.PagedCache(*x)
        values = [t.float() for t in x]
    slots = torch.randint(0, pages * page, (n,), device="cuda", generator=g).int()
    if n > 3:
        slots[0], slots[1], slots[2] = -1, pages * page, slots[3]
    inside = (slots >= 0) & (slots < pages * page)
    both = torch.full((n, 2, kv, hd), 5.5, device="cuda")
    D.paged_read(cache, slots, both[:, 0], both[:, 1])       # rows of one tensor
    alone = torch.full((n, kv, hd), 5.5, device="cuda")
    for i in (0, 1):
        want = values[i].reshape(-1, kv, hd)[slots.long().clamp(0, pages * page - 1)]
        want = torch.where(inside[:, None, None], want, 5.5)
        assert torch.equal(both[:, i], want)
        alone.fill_(5.5)
        D.paged_read(cache, slots, **{"kv"[i]: alone})
        assert torch.equal(alone, want)


def test_read_offsets_past_32_bits(gpu_ready):
    pages, page, kv, hd = 66000, 32, 8, 128     # 2.16e9 values each
    codes = [torch.empty(pages, page, kv, hd, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, kv, page, device="cuda") for _ in range(2)]
    cache = D.PagedCache(*codes, *scales)
    k, v = (torch.randn(2, kv, hd, device="cuda") for _ in range(2))
    last = ints([pages * page - 1, pages * page - page])
    D.paged_append(cache, k, v, None, last)
    back = [torch.empty(2, kv, hd, device="cuda") for _ in range(2)]
    D.paged_read(cache, last, *back)
    for x, y in zip((k, v), back):
        top = x.abs().amax(-1, keepdim=True)
        assert bool(((x - y).abs() <= top * (0.5 / 127 + 1e-6)).all())
    assert torch.equal(codes[0][-1, -1].double() * scales[0][-1, :, -1].double()[:, None],
                       back[0][0].double()) or torch.equal(
        codes[0][-1, -1].float() * scales[0][-1, :, -1][:, None], back[0][0])


# --------------------------------------------------------------- the attention

class Batch8(Batch):
    """Batch with its cache in codes; NaN scales wherever no sequence's key lies."""

    def __init__(self, seed, counts, lens, prefix, heads, kv, hd, page, **more):
        super().__init__(seed, counts, lens, prefix, heads, kv, hd, "f32", page, **more)
        g = torch.Generator(device="cuda").manual_seed(seed + 1)
        codes, scales = [], []
        for t in (self.keys, self.values):
            size = torch.exp(0.7 * torch.randn(*t.shape[:3], 1, device="cuda", generator=g))
            x = t * size
            top = x.abs().amax(-1)
            codes.append((127 * x / top[..., None]).nan_to_num(77.0 / 127).round().to(torch.int8))
            scales.append((top / 127).transpose(1, 2).contiguous())
        self.keys, self.values = codes
        self.key_scales, self.value_scales = scales
        self.take()

    def take(self):
        """The cache as it is now: the handle, and what each sequence's keys hold."""
        self.cache = D.PagedCache(self.keys, self.values, self.key_scales, self.value_scales)
        self.ws = D.paged_attention_workspace(self.cache, self.batch, self.heads)
        self.ws.fill_(0xff)

        def of(pages, count):
            pages = torch.from_numpy(np.asarray(pages[:-(-count // self.page)])).cuda().long()
            return [(c[pages].double() * s[pages].double().transpose(1, 2)[..., None])
                    .flatten(0, 1)[:count]
                    for c, s in ((self.keys, self.key_scales), (self.values, self.value_scales))]

        self.first_kv = of(self.shared, self.prefix)
        self.own_kv = [of(t, n) for t, n in zip(self.tables_h, self.kept_lens())]

    def kept_lens(self):
        return [o[0].shape[0] for o in self.own_kv]

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
            top = np.abs(v).max(-1)                    # 127 times the scale
            there = np.array([seen is None or seen(b, j) for j in range(len(k))], bool)
            for i in range(c):
                p = self.prefix + n - c + i
                j = np.arange(len(k))
                ok = there & (j <= p) & ((j > p - window) if window else True)
                for h in range(self.heads) if ok.any() else ():
                    kk, vv, tt = k[ok, h // group], v[ok, h // group], top[ok, h // group]
                    s = kk @ q[t, h] / np.sqrt(self.hd)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    e = (4 * U * np.abs(q[t, h]).max() * np.abs(kk).sum(1) / np.sqrt(self.hd)
                         + 8 * U * np.abs(s)).max() + 2 * U
                    of_step = maximum_filter1d(w * tt, 255, mode="constant")
                    want[t, h] = w @ vv
                    room[t, h] = ((2 * e + 2 * (len(kk) + 64) * U) * (w @ np.abs(vv))
                                  + 4 * U * (of_step / np.maximum(tt, 1e-300)) @ np.abs(vv))
                    if gate is not None:
                        g = 1 / (1 + np.exp(-gate[t, h]))
                        room[t, h] = (room[t, h] + 4 * U * np.abs(want[t, h])) * g
                        want[t, h] *= g
                t += 1
        return want, room


MORE = [
    # counts, lens, prefix, heads, kv, hd, page
    ([1], [64], 0, 4, 1, 128, 16), ([1], [65], 0, 4, 1, 64, 16), ([1], [257], 0, 20, 1, 128, 64),
    ([1] * 3, [255, 256, 1], 64, 32, 8, 128, 16), ([17], [300], 0, 4, 1, 128, 16),
    ([64, 65], [64, 300], 100, 4, 1, 64, 64), ([260], [900], 0, 8, 8, 128, 64),
    ([33, 1], [33, 800], 0, 4, 2, 128, 16), ([130], [520], 513, 6, 2, 64, 512),
]


@pytest.mark.parametrize("case", range(len(CASES + MORE)))
def test_attention(gpu_ready, case):
    counts, lens, prefix, heads, kv, hd, page = (CASES + MORE)[case]
    Batch8(case, counts, lens, prefix, heads, kv, hd, page, pad=case % 3, gate=case % 2 == 1).check()


@pytest.mark.parametrize("window", [1, 16, 50, 130, 512, 100000])
def test_window(gpu_ready, window):
    for counts, lens, prefix in (([1] * 4, [1, 40, 90, 600], 200), ([9, 30, 1], [9, 64, 300], 70),
                                 ([20], [150], 0), ([100, 3], [400, 700], 90)):
        Batch8(window, counts, lens, prefix, 6, 2, 64, 16, pad=1).check(window)
        Batch8(window, counts, lens, prefix, 8, 1, 128, 64).check(window)


@pytest.mark.parametrize("window", [0, 70, 700])
def test_many_sequences_of_unequal_lengths(gpu_ready, window):
    rng = np.random.default_rng(17)
    lens = rng.choice([0, 1, 5, 63, 64, 65, 128, 200, 333, 900], 130).tolist()
    counts = [min(int(c), max(n, 1)) for c, n in zip(rng.choice([0, 1, 1, 1, 2, 8], 130), lens)]
    Batch8(20, counts, lens, 100, 4, 2, 64, 16, pad=3, gate=True).check(window)
    one = [0] * 40 + [1] + [0] * 88 + [1]
    Batch8(21, one, [2000 if c else 0 for c in one], 0, 4, 2, 128, 64).check(window)
    Batch8(22, [1] * 64, list(range(64)), 0, 8, 4, 64, 16, max_len=100000).check(window)
    for seqs in (256, 257):
        lens = [int(n) for n in rng.integers(0, 40, seqs)]
        lens[3] = lens[-1] = 600
        Batch8(seqs, [1] * seqs, lens, 65, 2, 1, 64, 32).check(window)


def test_rows_without_keys_are_zeros(gpu_ready):
    b = Batch8(3, [1, 2, 1], [0, 1, 20], 0, 4, 2, 64, 16, pad=2)
    out = b.check()
    assert (out[0] == 0).all() and (out[1] == 0).all() and (out[2] != 0).any()
    b = Batch8(3, [1], [0], 0, 4, 2, 64, 16)
    assert (b.check() == 0).all()


@pytest.mark.parametrize("prefix", [1, 16, 63, 64, 65, 128, 250])
def test_short_prefix(gpu_ready, prefix):
    for (heads, kv, hd, page), counts in itertools.product(
            [(2, 2, 64, 16), (6, 2, 128, 64), (8, 1, 64, 32)], [[1, 1, 0, 1], [3, 1, 2, 0]]):
        b = Batch8(prefix, counts, [60, 1, 33, 4], prefix, heads, kv, hd, page, pad=1, gate=True)
        for window in (0, 1, 5, 40, 64, prefix, prefix + 1, 100, 1000):
            b.check(window)
        b.batch.prefix_pages[-1] = -1
        b.tables[0, 0] = 0x7fffffff
        last = (prefix - 1) // page * page
        b.check(seen=lambda s, j: j < last if j < prefix else s != 0 or j - prefix >= page)


@pytest.mark.parametrize("counts,lens,prefix,heads,hd", [
    ([1], [70001], 0, 2, 64), ([2, 1], [33000, 5], 40000, 3, 64), ([1], [20], 66000, 9, 128)])
def test_many_runs(gpu_ready, counts, lens, prefix, heads, hd):
    b = Batch8(13, counts, lens, prefix, heads, 1, hd, 256, pad=1, gate=True)
    b.check()
    b.check(3000)


def test_two_calls_at_once(gpu_ready):
    make = lambda: Batch8(12, [1] * 9, [40 * i + 1 for i in range(9)], 700, 8, 4, 64, 32)
    a, b = make(), make()
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


def test_more_tokens_than_own_keys(gpu_ready):
    for count, own, prefix in ((3, 1, 50), (70, 66, 0), (100, 3, 300), (6, 0, 900)):
        b = Batch8(9, [count, 1], [own, 2000], prefix, 4, 2, 64, 16)
        want, room = b.expected()
        rest = count - own
        for window in (0, 5000, 0x7fffffff):
            out = host(b.run(window))
            assert (np.abs(out[rest:] - want[rest:]) <= room[rest:]).all()
            if prefix == 0:
                assert (out[:rest] == 0).all()
                continue
            for i in range(0, rest, 7):
                alone = Batch8(9, [1], [0], prefix, 4, 2, 64, 16)
                alone.first_kv = b.first_kv
                alone.q.copy_(b.q[i:i + 1])
                got, bound = alone.expected()
                assert (np.abs(out[i] - got[0]) <= bound[0]).all(), (window, i)


@pytest.mark.parametrize("prefix", [40, 500])
@pytest.mark.parametrize("counts", [[1, 1], [1, 5], [70, 2]])
def test_a_window_far_behind_the_keys(gpu_ready, counts, prefix):
    b = Batch8(15, counts, [60, 20], prefix, 4, 2, 64, 16)
    for far in (1 << 20, 0x7fffffff - prefix, 0x7fffffff):
        b.lens_d.fill_(far)
        for window in (1, 50, 100000):
            assert (host(b.run(window)) == 0).all(), (far, window)


@pytest.mark.parametrize("heads,kv,seqs,tokens,most,page,width,prefix", [
    (8, 8, 4096, 4200, 4200, 64, 290, 0), (8, 8, 4096, 4200, 4200, 64, 290, 300),
    (16, 16, 65536, 2000, 20, 256, 71, 0), (4, 1, 50000, 4200, 4200, 256, 70, 40)])
def test_bounds_far_above_the_batch(gpu_ready, heads, kv, seqs, tokens, most, page, width, prefix):
    counts, lens = [19, 1, 7, 2, 20], [40, 600, 7, 1, 333]
    if most > 100:
        counts[0], lens[0] = 150, 180
    b = Batch8(17, counts, lens, prefix, heads, kv, 64, page, pad=5, gate=True)
    rng = np.random.default_rng(seqs)
    at = np.sort(rng.permutation(np.arange(1, seqs - 1))[:3])
    at = np.concatenate([[0], at, [seqs - 1]])
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


@pytest.mark.parametrize("window", [0, 90])
def test_a_prompt_among_single_tokens(gpu_ready, window):
    counts = [1] * 40 + [210] + [1, 0, 3, 17] * 8
    lens = [max(c, 5 * i + 1) for i, c in enumerate(counts)]
    Batch8(31, counts, lens, 0, 8, 4, 64, 16, pad=2, gate=True).check(window)
    Batch8(32, counts, lens, 300, 4, 4, 64, 32, pad=70).check(window)
    short = [min(c, 17) for c in counts]
    Batch8(33, short, lens, 0, 64, 32, 64, 64).check(window)
    Batch8(34, [900, 300], [900, 400], 0, 6, 1, 64, 64, pad=1).check(window)


@pytest.mark.parametrize("prefix", [0, 32, 500])
def test_lengths_past_the_bound(gpu_ready, prefix):
    b = Batch8(18, [1, 2], [100, 48], prefix, 4, 2, 64, 16)
    b.lens = [1 << 30, 1 << 30]
    b.lens_d.copy_(ints(b.lens))
    out = b.check().copy()
    b.lens_d.copy_(ints([100, 1000]))
    assert np.array_equal(out, host(b.run()))


def test_pages_outside_the_cache_are_not_seen(gpu_ready):
    b = Batch8(4, [1, 3], [100, 90], 64, 8, 4, 128, 16)
    b.tables[0, 2], b.tables[1, 0] = -1, b.keys.shape[0]
    b.tables[1, 3] = 0x7fffffff
    missing = {0: [2], 1: [0, 3]}
    b.check(seen=lambda s, j: j < 64 or (j - 64) // 16 not in missing[s])
    b.tables.fill_(-1)
    b.check(seen=lambda s, j: j < 64)
    b = Batch8(5, [2], [40], 0, 2, 2, 64, 32)
    b.tables.fill_(1 << 30)
    assert (host(b.run()) == 0).all()
    b = Batch8(5, [90], [200], 0, 2, 2, 64, 16)         # blocks of 64 rows
    b.tables[0, 3] = -5
    b.check(seen=lambda s, j: j // 16 != 3)


@pytest.mark.parametrize("heads,kv,hd,page", [(4, 2, 64, 16), (64, 2, 64, 64), (64, 1, 128, 16),
                                              (64, 1, 128, 128)])
def test_nan_behind_the_mask(gpu_ready, heads, kv, hd, page):
    """A scale of NaN or infinity at a later token's place does not reach the
    earlier ones; a head that sees it is no finite number, but for scores of
    -infinity, whose key then has no weight."""
    make = lambda: Batch8(8, [6], [40], 50, heads, kv, hd, page)
    want, room = make().expected()
    without, room_without = make().expected(seen=lambda s, j: j != 50 + 37)
    for what in ("key_scales", "value_scales"):
        for bad in (np.inf, -np.inf, np.nan):
            b = make()
            j = 37                                  # seen by tokens 3, 4 and 5 (places 37 .. 39)
            getattr(b, what)[int(b.tables_h[0, j // page]), 0, j % page] = bad
            out = host(b.run())
            assert (np.abs(out[:3] - want[:3]) <= room[:3]).all(), (what, bad)
            hit = np.s_[3:, :heads // kv]
            right = ~np.isfinite(out[hit])
            if what == "key_scales" and np.isinf(bad):
                right |= np.abs(out[hit] - without[hit]) <= room_without[hit]
                q = b.q[hit].double().cpu().numpy()
                code = b.keys[int(b.tables_h[0, j // page]), j % page, 0].double().cpu().numpy()
                assert (np.isnan(out[hit]).all(-1) == (q @ code * bad > 0)).all()
            assert right.all(), (what, bad)
            rest = np.s_[3:, heads // kv:]
            assert (np.abs(out[rest] - want[rest]) <= room[rest]).all()
    b = make()
    want, room = b.expected(60)
    for t in (b.key_scales, b.value_scales):
        t[int(b.shared[0]), :, :2] = float("nan")
    assert (np.abs(host(b.run(60)) - want) <= room).all()
    b = make()
    b.q[1, 0, 3], b.q[2, 0, 5] = float("inf"), float("nan")
    out = host(b.run())
    assert np.isnan(out[1:3, 0]).all()
    want, room = make().expected()
    assert (np.abs(out - want) <= room)[[0, 3, 4, 5]].all()


def test_weights_of_nothing_and_much(gpu_ready):
    """Scales of zero, of very different sizes within a step, and very small and
    very large ones; scores of thousands."""
    Batch8(10, [1, 4], [70, 80], 130, 8, 2, 128, 16, scale=300.0).check()
    for scale in (0.0, 1e-6, 1e6):
        b = Batch8(40, [1, 40], [300, 90], 77, 8, 2, 64, 32)
        b.value_scales[..., ::3] *= scale
        b.take()
        b.check()
    for by in (1e-25, 1e25):
        b = Batch8(41, [1, 40], [300, 90], 77, 8, 2, 64, 32)
        b.value_scales *= by
        b.take()
        b.check()
        b = Batch8(41, [1, 40], [300, 90], 77, 8, 2, 64, 32)
        b.key_scales *= by
        b.q /= by
        b.take()
        b.check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("counts", [[1, 3], [150]])
def test_next_to_powers_of_two(gpu_ready, counts, hd):
    """Queries and weights whose digits are the largest there are: values at a
    power of two, next to it, and some thousandths below it."""
    edges = np.float32([1, -1, np.nextafter(np.float32(1), np.float32(0)),
                        -np.nextafter(np.float32(1), np.float32(0)), 0.9925, -0.9925, 0.9921, -0.9921,
                        0.998, -0.9999, 1 + 2.0 ** -23, 0.5, -0.25])
    rng = np.random.default_rng(hd)
    for fill in (1.0, 0.05):
        b = Batch8(43, counts, [200, 90][:len(counts)], 70, 8, 2, hd, 32)
        q = rng.choice(edges, tuple(b.q.shape)) * np.where(rng.random(tuple(b.q.shape)) < fill, 1, 0.1)
        q *= 2.0 ** rng.integers(-3, 2, (*b.q.shape[:2], 1))
        b.q.copy_(torch.from_numpy(q.astype(np.float32)))
        b.value_scales.copy_(torch.from_numpy(np.abs(rng.choice(edges, tuple(b.value_scales.shape)))))
        b.keys.copy_((b.keys.float() / 16).round().to(torch.int8))     # weights of nearly one
        b.take()
        b.check()


def test_far_tail(gpu_ready):
    """One key that outweighs every other, and a long tail that together weighs
    as much: none of it is lost."""
    b = Batch8(42, [1], [20000], 0, 2, 1, 64, 64)
    b.q.zero_()
    b.q[..., 0] = 8.0
    b.keys.fill_(0)
    page = int(b.tables_h[0, 0])
    b.keys[page, 5, :, 0] = 127
    b.key_scales.fill_(float(np.log(20000.0) / 127))       # a score of log 20000 against zeros
    b.values[:, :, :, :] = b.values.abs()
    b.take()
    b.check()


def test_offsets_past_32_bits(gpu_ready):
    pages, page, kv, hd = 66000, 32, 8, 128     # 2.16e9 codes each
    keys, values = (torch.empty(pages, page, kv, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(pages, kv, page, device="cuda") for _ in range(2))
    for counts in ([1, 2], [70, 2]):
        small = Batch8(11, counts, [90, 70], 40, 8, 8, 128, 32)
        want = host(small.run()).copy()
        shift = pages - small.keys.shape[0]
        for t, s in ((keys, small.keys), (values, small.values), (ks, small.key_scales),
                     (vs, small.value_scales)):
            t[shift:] = s
        batch = D.PagedBatch(small.starts, small.lens_d, small.tables + shift, small.live,
                             max(counts), 90, prefix_pages=ints(small.shared + shift), prefix_len=40)
        out = torch.empty_like(small.out)
        D.paged_attention(D.PagedCache(keys, values, ks, vs), batch, small.q, out, small.ws)
        assert np.array_equal(host(out), want)


def test_same_bits_again_on_another_stream(gpu_ready):
    b = Batch8(12, [1] * 20, list(range(30, 230, 10)), 1000, 16, 4, 128, 32)
    first = b.run().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b.out.fill_(0)
    side.wait_stream(torch.cuda.current_stream())
    b.run(stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(b.out, first)


def test_most_rows(gpu_ready):
    """As many rows as a call may have, nearly all of them padding."""
    rows, heads, kv = 1082401, 62, 31             # 2^26 - 2 rows of the result
    b = Batch8(14, [3], [40], 500, heads, kv, 64, 16)
    batch = D.PagedBatch(b.starts, b.lens_d, b.tables, rows, 3, 40,
                         prefix_pages=b.batch.prefix_pages, prefix_len=500)
    ws = D.paged_attention_workspace(b.cache, batch, heads)
    q, out = (torch.empty(rows, heads, 64, device="cuda") for _ in range(2))
    q[:3] = b.q
    out.fill_(3.25)
    D.paged_attention(b.cache, batch, q, out, ws)
    want, room = b.expected()
    assert (np.abs(host(out[:3]) - want) <= room).all()
    assert not bool((out[3:] != 3.25).any())


def test_steps_to_tokens_eager_and_captured(gpu_ready):
    """Decode steps as a server runs them: append, attention, the int8 rows of its
    output, their product with a head of 3001 tokens, and a token for each
    sequence, over growing sequences; once eagerly and once as one captured graph
    whose arrays change, with the program's own work between the replays. The
    prefix is read back and written to another cache, which holds the same."""
    seqs, prefix, heads, kv, hd, page, steps, vocab = 5, 75, 8, 2, 64, 16, 6, 3001
    rows, width = seqs + 3, 6
    rng = np.random.default_rng(13)
    g = torch.Generator(device="cuda").manual_seed(13)
    pages = 8 + seqs * width
    order = rng.permutation(pages).astype(np.int32)
    shared, tables_h = order[:5], order[5:5 + seqs * width].reshape(seqs, width)
    rope = torch.from_numpy(rope_table(512, hd)).cuda()
    w = 1 + 0.1 * torch.randn(hd, device="cuda", generator=g)
    head = torch.randn(vocab, heads * hd, device="cuda", generator=g)
    head_q = torch.empty(vocab, heads * hd, dtype=torch.int8, device="cuda")
    head_s = torch.empty(vocab, device="cuda")
    D.quantize_i8r(head, head_q, head_s, vocab, heads * hd, heads * hd)
    step_qkv = [torch.randn(rows, (heads + 2 * kv) * hd, device="cuda", generator=g)
                for _ in range(steps)]
    step_u = torch.rand(steps, rows, device="cuda", generator=g)
    par = [torch.tensor(x, device="cuda") for x in ([0.9, 1.0, 0.0, 1.2, 0.7, 1.0, 1.0, 1.0],
                                                    [0.9, 1.0, 1.0, 0.95, 0.5, 1.0, 1.0, 1.0])]
    top_k = ints([40, 0, 0, 200, 0, 0, 0, 0])
    begin = [3, 17, 40, 15, 60]
    history = [torch.randn(n, 2 * kv * hd, device="cuda", generator=g) for n in [prefix] + begin]

    def play(captured):
        kept = empty_cache(pages, page, kv, hd)
        cache = D.PagedCache(*kept)
        for i, x in enumerate(history):     # prompts, appended many tokens at once
            n = x.shape[0]
            table = shared if i == 0 else tables_h[i - 1]
            own = np.arange(n)
            D.paged_append(cache, x[:, :kv * hd].view(n, kv, hd), x[:, kv * hd:].view(n, kv, hd),
                           ints(own + (0 if i == 0 else prefix)),
                           ints(table[own // page] * page + own % page), rope=rope, k_norm=w)
        starts, lens, tables = ints(list(range(seqs + 1))), ints(begin), ints(tables_h)
        positions, slots = ints([0] * rows), ints([-1] * rows)
        qkv = torch.empty(rows, (heads + 2 * kv) * hd, device="cuda")
        q = qkv[:, :heads * hd].view(rows, heads, hd)
        k = qkv[:, heads * hd:(heads + kv) * hd].view(rows, kv, hd)
        v = qkv[:, (heads + kv) * hd:].view(rows, kv, hd)
        q_rot, out = (torch.zeros(rows, heads, hd, device="cuda") for _ in range(2))
        out_q = torch.empty(rows, heads * hd, dtype=torch.int8, device="cuda")
        out_s, u = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        logits = torch.empty(rows, vocab, device="cuda")
        tokens = torch.full((rows,), -9, dtype=torch.int32, device="cuda")
        batch = D.PagedBatch(starts, lens, tables, rows, 1, width * page, prefix_pages=ints(shared),
                             prefix_len=prefix)
        ws, sample_ws = D.paged_attention_workspace(cache, batch, heads), D.sample_workspace(rows, vocab)

        def step():
            D.paged_append(cache, k, v, positions, slots, rope=rope, q=q, q_out=q_rot, q_norm=w,
                           k_norm=w)
            D.paged_attention(cache, batch, q_rot, out, ws)
            D.quantize_i8r(out, out_q, out_s, rows, heads * hd, heads * hd)
            D.gemm_i8r(head_q, head_s, out_q, out_s, logits, vocab, heads * hd, rows)
            D.sample(logits, u, tokens, sample_ws, temperature=par[0], top_k=top_k, top_p=par[1])

        graph, got = None, []
        for i in range(steps):
            at = np.array(begin) + i
            lens.copy_(ints(at + 1))
            positions[:seqs] = ints(prefix + at)
            slots[:seqs] = ints(tables_h[np.arange(seqs), at // page] * page + at % page)
            qkv.copy_(step_qkv[i])
            u.copy_(step_u[i])
            if captured:
                if graph is None:           # capture runs nothing
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        step()
                graph.replay()
            else:
                step()
            got.append((out.clone(), logits.clone(), tokens.clone()))
            torch.cuda.synchronize()
        return cache, kept, q_rot.clone(), got

    cache, kept, q_rot, eager = play(False)
    _, kept2, _, replayed = play(True)
    for a, b in zip(eager, replayed):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert all(torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0)) for x, y in zip(kept, kept2))
    # Each step's tokens against the definition on its logits.
    for i, (_, logits, tokens) in enumerate(eager):
        for r in range(seqs):
            want = answers(host(logits[r]), float(step_u[i, r]), float(par[0][r]), int(top_k[r]),
                           float(par[1][r]), 0.0)
            assert int(tokens[r]) in want, (i, r)
    # The last step's attention against the formula on what the cache holds.
    flat = [stored(kept[j], kept[2 + j]) for j in (0, 1)]
    q = q_rot.double().cpu().numpy()
    for b in range(seqs):
        n = begin[b] + steps
        places = np.concatenate([shared[np.arange(prefix) // page] * page + np.arange(prefix) % page,
                                 tables_h[b][np.arange(n) // page] * page + np.arange(n) % page])
        kk, vv = flat[0][places], flat[1][places]
        assert np.isfinite(kk).all() and np.isfinite(vv).all()
        for h in range(heads):
            k1, v1 = kk[:, h // 4], vv[:, h // 4]
            s = k1 @ q[b, h] / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            e = (4 * U * np.abs(q[b, h]).max() * np.abs(k1).sum(1) / np.sqrt(hd) + 8 * U * np.abs(s)).max() + 2 * U
            top = np.abs(v1).max(1)
            of_step = maximum_filter1d(p * top, 255, mode="constant")
            room = (2 * e + 2 * (len(k1) + 64) * U) * (p @ np.abs(v1)) + 4 * U * (of_step / top) @ np.abs(v1)
            assert (np.abs(eager[-1][0][b, h].double().cpu().numpy() - p @ v1) <= room).all()
    # The prefix moved to another cache: read back, appended, the same again.
    at = ints(shared[np.arange(prefix) // page] * page + np.arange(prefix) % page)
    back = [torch.empty(prefix, kv, hd, device="cuda") for _ in range(2)]
    D.paged_read(cache, at, *back)
    other = D.PagedCache(*empty_cache(pages, page, kv, hd))
    D.paged_append(other, *back, None, at)
    again = [torch.empty(prefix, kv, hd, device="cuda") for _ in range(2)]
    D.paged_read(other, at, *again)
    for x, y in zip(back, again):          # the largest code is 127 again: its scale moves by a rounding
        assert bool(((x - y).abs() <= 2 * U * x.abs()).all())


def test_refusals(gpu_ready):
    k, v, ks, vs = empty_cache(4, 16, 2, 64)
    for bad in ((k, v), (k, v, ks, None), (k, v, ks[:, :1], vs), (k, v, ks.double(), vs.double()),
                (k, v.float(), ks, vs), (k.float(), v.float(), ks, vs), (k, v, ks.cpu(), vs),
                (k, v, ks.transpose(0, 1).contiguous().transpose(0, 1), vs)):
        with pytest.raises(ValueError):
            D.PagedCache(*bad)
    with pytest.raises(RuntimeError):       # not 16-byte aligned
        odd = torch.empty(4 * 2 * 16 + 1, device="cuda")[1:].view(4, 2, 16)
        D.paged_read(D.PagedCache(k, v, odd, vs), ints([0]), torch.empty(1, 2, 64, device="cuda"))
    cache = D.PagedCache(k, v, ks, vs)
    out = torch.empty(3, 2, 64, device="cuda")
    for slots, a in ((ints([0, 1]), out), (ints([0, 1, 2]).long(), out), (ints([0, 1, 2]), out.double()),
                     (ints([0, 1, 2]), out[:, :1]), (ints([0, 1, 2]), out.cpu()),
                     (ints([0, 1, 2]), out.view(3, 128)), (ints([0, 1, 2]).cpu(), out)):
        with pytest.raises(ValueError):
            D.paged_read(cache, slots, a)
    with pytest.raises(RuntimeError):
        D.paged_read(cache, ints([0, 1, 2]))
