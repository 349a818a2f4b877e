"""A small top_k over vocabularies past a quarter of a million ids, where a row has more waves than a wave can rank."""
import time

import numpy as np
import pytest

from test_gpu_kv8 import Bufs
from test_gpu_operator_aliases import Alias
from test_gpu_sample import check, rows_of, sample, settings

pytestmark = pytest.mark.gpu


def least_us(gpu, x, sets):
    """The shortest of 30 calls, all buffers on the device."""
    rows, vocab = x.shape
    with Bufs(gpu) as buf:
        b = [buf(a) for a in (x, settings(sets), np.full(rows, 0.37, np.float32), np.zeros(rows, np.uint32))]
        h = [Alias(gpu, a, a.nbytes) for a in b]
        gpu.sample(b[0], b[1], b[2], b[3], None, [vocab, rows])         # sends them
        t = []
        for _ in range(30):
            t0 = time.perf_counter()
            gpu.sample(h[0], h[1], h[2], h[3], None, [vocab, rows])
            t.append(time.perf_counter() - t0)
        for a in h:
            a.free()
    return 1e6 * min(t)


def test_a_small_top_k_costs_no_more_than_a_larger_one(gpu):
    """It was four times as much at a million ids."""
    x = rows_of(np.random.default_rng(1), 1, 1000000)
    other = least_us(gpu, x, [(0.7, 140, 0.8, 0.0)])
    for s in ((0.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0)):
        t = least_us(gpu, x, [s])
        assert t < 2.5 * other, (s, t, other)


@pytest.mark.parametrize("vocab,rows", [(262144, 1), (262145, 1), (262145, 2), (530001, 1), (1048577, 1), (300000, 3)])
@pytest.mark.parametrize("coarse", [False, True])
def test_small_top_k_over_large_vocabularies(gpu, vocab, rows, coarse):
    rng = np.random.default_rng(vocab + coarse)
    x = rows_of(rng, rows, vocab, coarse)
    for s in ((0.0, 0, 1.0, 0.0), (1.0, 1, 0.5, 0.0), (0.8, 20, 1.0, 0.0), (1.0, 128, 0.93, 0.01), (0.7, 50, 0.8, 0.0)):
        tok, _ = check(gpu, x, [s] * rows, np.full(rows, 0.4321))
        again, _ = sample(gpu, x, [s] * rows, np.full(rows, 0.4321), probs=False)
        assert np.array_equal(tok, again)
