"""dnx_sample_workspace_bytes: a workspace for the most rows and the largest vocabulary
serves every call of less."""

import random

from dianoia_amd import _lib


def test_size_never_falls():
    size = _lib.load().dnx_sample_workspace_bytes
    for vocab in (1, 700, 8192, 8193, 9000, 32003, 128000, 131077, 151936, 262145, 1 << 20):
        sizes = [size(rows, vocab) for rows in list(range(1, 1500)) + [4096, 65535, 65536]]
        assert sizes == sorted(sizes), vocab
    for rows in (1, 2, 5, 9, 54, 64, 257, 1025, 65536):
        sizes = [size(rows, vocab) for vocab in [*range(1, 200000, 61), *range(200000, (1 << 20) + 1, 509)]]
        assert sizes == sorted(sizes), rows
    rng = random.Random(1)
    for _ in range(20000):
        rows, vocab = rng.randint(1, 2000), int(2 ** rng.uniform(0, 20))
        assert size(rng.randint(1, rows), rng.randint(1, vocab)) <= size(rows, vocab)
