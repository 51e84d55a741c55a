"""dnx_paged_attention over int8 caches where blocks of 64 rows are taken: many new
tokens of few keys, and prefixes that many rows over few key heads share. Bounds as in
test_gpu_paged_i8_range.py; test_paged_split_i8_wide.py says that these shapes take
them."""

import numpy as np
import pytest
import torch

from dianoia_amd import device as D
from gpu_util import host
from test_gpu_paged import ints
from test_gpu_paged_i8_range import Tight, times

pytestmark = pytest.mark.gpu


def ragged(seqs, most, tokens, seed):
    """Lengths up to `most` with borders of steps among them; one new token in every
    sixth sequence, about `tokens` in the others."""
    rng = np.random.default_rng(seed)
    lens = rng.choice([63, 64, 65, 100, 127, 128, 129, most - 1, most, most], seqs)
    lens = np.minimum(lens, most)
    counts = np.minimum([1 if i % 6 == 5 else tokens - i % 2 for i in range(seqs)], lens)
    lens[0], counts[0], lens[-1], counts[-1] = most, min(tokens, most), 1, 1
    return counts.tolist(), lens.tolist()


# counts, lens, prefix, heads, kv, page
OWN = [(*ragged(48, 190, 45, 1), 0, 8, 8, 16), (*ragged(60, 200, 25, 2), 0, 12, 4, 32),
       (*ragged(24, 190, 100, 3), 70, 8, 8, 64), (*ragged(160, 190, 12, 4), 300, 8, 2, 16),
       (*ragged(3, 130, 130, 5), 0, 64, 32, 64)]
PREFIX = [([1] * 257, [1 + i % 40 for i in range(257)], 100, 4, 1, 16), ([260, 3], [290, 200], 65, 4, 1, 64),
          ([37, 1, 100, 0, 128], [40, 9, 100, 7, 500], 2100, 8, 2, 32), ([1] * 350, [3] * 350, 1, 9, 3, 16),
          ([130] * 3, [130, 200, 400], 640, 12, 4, 128)]
SHAPES = OWN + PREFIX
BOUNDED = [190] * 4 + [1] * 60 + [2, 0, 33], [190] * 4 + [3 * i + 1 for i in range(60)] + [7, 0, 180]


def batch(seed, i, hd, **more):
    counts, lens, prefix, heads, kv, page = SHAPES[i]
    return Tight(seed, counts, lens, prefix, heads, kv, hd, page, **more)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(gpu_ready, shape, hd):
    b = batch(shape, shape, hd, pad=shape % 3, gate=shape % 2 == 1)
    b.check()
    b.check(100)
    b.check(1)


@pytest.mark.parametrize("hd", [64, 128])
def test_queries_of_every_size(gpu_ready, hd):
    rng = np.random.default_rng(hd)
    for shape in (1, 3, 5, 6):
        b = batch(70, shape, hd)
        rows = tuple(b.q.shape[:2])
        times(b.q, rng.integers(-155, 4, rows)[..., None])
        b.q[torch.from_numpy(rng.random(rows) < 0.1)] = 0.0
        b.check()
        b = batch(71, shape, hd)
        times(b.key_scales, 105)
        times(b.q, rng.integers(-120, -98, rows)[..., None])
        b.take()
        b.check()
        b = batch(72, shape, hd)
        b.q[..., 5] *= 3000.0
        b.keys[..., 5] = 0
        b.take()
        b.check()


@pytest.mark.parametrize("hd", [64, 128])
def test_pages_outside_the_cache_are_not_seen(gpu_ready, hd):
    b = batch(73, 0, hd)
    b.tables[0, 2], b.tables[3, 0], b.tables[7, 1] = -1, b.keys.shape[0], 0x7fffffff
    missing = {0: 2, 3: 0, 7: 1}
    b.check(seen=lambda s, j: j // 16 != missing.get(s, -1))
    b = batch(74, 7, hd)
    b.batch.prefix_pages[3] = -5
    b.check(seen=lambda s, j: j >= 2100 or j // 32 != 3)
    b.check(300, seen=lambda s, j: j >= 2100 or j // 32 != 3)
    b.batch.prefix_pages.fill_(1 << 30)
    b.check(seen=lambda s, j: j >= 2100)


@pytest.mark.parametrize("hd", [64, 128])
def test_nan_behind_the_mask(gpu_ready, hd):
    """Scales of NaN at a sequence's last key: the rows before it do not change."""
    for shape in (0, 3):
        b = batch(75, shape, hd)
        want, room = b.expected()
        page, t, hit = b.page, 0, np.zeros(b.live, bool)
        for s, (c, n) in enumerate(zip(b.counts, b.lens)):
            at = (int(b.tables_h[s, (n - 1) // page]), slice(None), (n - 1) % page)
            b.key_scales[at] = b.value_scales[at] = float("nan")
            hit[t + c - 1] = c > 0
            t += c
        out = host(b.run())[:b.live]
        assert np.isnan(out[hit]).all()
        assert (np.abs(out - want) <= room)[~hit].all()


def test_next_to_powers_of_two(gpu_ready):
    edges = np.float32([1, -1, np.nextafter(np.float32(1), np.float32(0)), 0.9925, -0.9921, 0.998, -0.9999,
                        1 + 2.0 ** -23, 0.5, -0.25])
    rng = np.random.default_rng(3)
    for shape in (1, 5):
        b = batch(76, shape, 128)
        q = rng.choice(edges, tuple(b.q.shape)) * 2.0 ** rng.integers(-3, 2, (*b.q.shape[:2], 1))
        b.q.copy_(torch.from_numpy(q.astype(np.float32)))
        b.value_scales.copy_(torch.from_numpy(np.abs(rng.choice(edges, tuple(b.value_scales.shape)))))
        b.keys.copy_((b.keys.float() / 16).round().to(torch.int8))     # weights of nearly one
        b.take()
        b.check()


@pytest.mark.parametrize("window", [0, 70])
def test_bounds_above_the_batch(gpu_ready, window):
    """Every sequence might have as many tokens and keys as the largest: its blocks lie in
    a row, and most runs hold no key."""
    counts, lens = BOUNDED
    b = Tight(77, counts, lens, 0, 16, 8, 64, 16, pad=3)
    b.batch = D.PagedBatch(b.starts, b.lens_d, b.tables, b.live + 3, 700, 190)
    b.ws = D.paged_attention_workspace(b.cache, b.batch, b.heads)
    b.ws.fill_(0xff)
    b.check(window)


def test_captured_with_other_lengths_at_each_replay(gpu_ready):
    b = batch(78, 0, 128, gate=True)
    first = b.run().clone()
    torch.cuda.synchronize()
    lens = list(b.lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.run()
    for i in range(4):
        b.lens = [max(n - 7 * i, c) for n, c in zip(lens, b.counts)]
        b.lens_d.copy_(ints(b.lens))
        b.out.fill_(3.25)
        graph.replay()
        torch.cuda.synchronize()
        got = b.out.clone()
        assert torch.equal(got, b.run())
        if i == 0:
            assert torch.equal(got, first)
        want, room = b.expected()
        assert (np.abs(host(got)[:b.live] - want) <= room).all()
