"""A small top_k over few waves of ids: vocabularies and masks that leave fewer of them than top_k wants, or hardly more."""
import time

import numpy as np
import pytest

import pages_oracle as P
from test_gpu_kv8 import Bufs
from test_gpu_operator_aliases import Alias
from test_gpu_sample import check, rows_of, sample, settings

pytestmark = pytest.mark.gpu


def masked(rng, vocab, first, n, step=1):
    x = rows_of(rng, 1, vocab)
    y = np.full_like(x, -np.inf)
    y[:, first:first + n * step:step] = x[:, first:first + n * step:step]
    return y


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


def logits_of(kind):
    rng = np.random.default_rng(9)
    return rows_of(rng, 1, kind) if isinstance(kind, int) else masked(rng, *kind)


@pytest.mark.parametrize("kind,ks", [(4099, (18, 20, 24)), (32000, (126, 128)), ((151936, 5000, 4096), (18, 50, 128)), ((600000, 77777, 9000), (50, 100))])
def test_no_row_goes_to_one_workgroup_for_want_of_waves(gpu, kind, ks):
    """A small top_k costs about what a larger one does, which has a form of its own, whatever the waves leave (it was 4 to 30 times
    as much where fewer waves had ids than top_k)."""
    x = logits_of(kind)
    other = least_us(gpu, x, [(0.7, 140, 0.8, 0.0)])
    for k in ks:
        t = least_us(gpu, x, [(0.7, k, 0.8, 0.0)])
        assert t < 2.5 * other, (k, t, other)


KINDS = [2049, 2100, 4099, 10000, 32000, 32001, (151936, 5000, 4096), (151936, 5000, 2049), (151936, 5000, 2048), (151936, 250, 12), (151936, 7, 13, 11000),
         (151936, 0, 3000, 50), (300000, 77777, 9000), (600000, 599000, 1000), (600000, 100, 30000)]


@pytest.mark.parametrize("kind", KINDS)
def test_small_top_k_over_few_waves(gpu, kind):
    rng = np.random.default_rng(10)
    x = logits_of(kind)
    ks = [1, 2, 8, 12, 13, 15, 16, 17, 18, 24, 25, 36, 37, 50, 100, 124, 125, 126, 127, 128, 129]
    for p, m in ((1.0, 0.0), (0.83, 0.0), (0.97, 0.02)):
        sets = [(0.9, k, p, m) for k in ks]
        tok, _ = check(gpu, np.repeat(x, len(ks), 0), sets, np.full(len(ks), 0.7312))
        again, _ = sample(gpu, np.repeat(x, len(ks), 0), sets, np.full(len(ks), 0.7312), probs=False)
        assert np.array_equal(tok, again)
    for k in (17, 126):         # one row: the parts are smaller
        check(gpu, x, [(1.3, k, 0.9, 0.0)], rng.random(1))
        check(gpu, x, [(1.3, k, 0.9, 0.0)], rng.random(1), in_place=True)


def test_rows_of_both_kinds_together(gpu):
    """The same top_k over rows of which some have enough waves, some too few, some nothing at all; ids alike in the rest."""
    rng = np.random.default_rng(11)
    v = 151936
    x = np.concatenate([rows_of(rng, 1, v), masked(rng, v, 5000, 4096), np.full((1, v), -np.inf, np.float32), masked(rng, v, 9, 5), rows_of(rng, 1, v, True),
                        masked(rng, v, 100000, 3000)])
    x[5, 100000:103000] = np.round(x[5, 100000:103000])
    for s in ((0.8, 50, 0.9, 0.0), (1.0, 100, 1.0, 0.01)):
        check(gpu, x, [s] * 6, rng.random(6))
        tok, _ = sample(gpu, x, [s] * 6, [0.4] * 6, probs=False)
        assert tok[2] == 0xFFFFFFFF


@pytest.mark.parametrize("rows,vocab,left", [(140, 60000, 20000), (140, 60003, 3000), (1100, 9000, 4000)])
def test_many_rows_over_few_waves(gpu, rows, vocab, left):
    """Parts of several rounds, and more rows than go at once; a mask that leaves `left` ids in a row, another place in each row."""
    rng = np.random.default_rng(vocab)
    x = (2 * rng.standard_normal((rows, vocab))).astype(np.float32)
    for r in range(rows):
        first = int(rng.integers(0, vocab - left))
        x[r, :first] = x[r, first + left:] = -np.inf
    sets = [(0.9, (20, 37, 40, 64)[r % 4], (0.9, 1.0)[r % 3 == 0], 0.0) for r in range(rows)]
    u = rng.random(rows).astype(np.float32)
    tok, pr = sample(gpu, x, sets, u)
    again, _ = sample(gpu, x, sets, u, probs=False)
    assert np.array_equal(tok, again)
    for r in np.unique(np.concatenate([np.arange(8), rng.integers(0, rows, 12), [min(1023, rows - 1), min(1024, rows - 1), rows - 1]])):
        want, probs, margin = P.sample(x[r], *sets[r], u[r])
        assert margin > 1e-11 and int(tok[r]) == want
        assert (np.abs(pr[r] - probs) <= probs * (2.0 ** -24 + 1e-9) + 2.0 ** -149).all()
        assert np.array_equal(pr[r] > 0, probs.astype(np.float32) > 0)
