"""The forms that sampling takes by size and settings: lists of few ids and of thousands, top-k and top-p borders each
alone and together, lists that do not fit, several rounds a part, more rows than go at once."""
import numpy as np
import pytest

import pages_oracle as P
from test_gpu_sample import check, sample

pytestmark = pytest.mark.gpu


def crowd(rng, v, n, width=1e-3):
    """A few ids high up, n ids within `width` of each other, the rest far below."""
    x = (-12 + rng.random(v)).astype(np.float32)
    at = rng.permutation(v)
    x[at[:n]] = (4 + width * rng.random(n)).astype(np.float32)
    x[at[n:n + 6]] = (6 + rng.random(6)).astype(np.float32)
    return x


@pytest.mark.parametrize("n", [3, 60, 64, 65, 120, 128, 129, 500, 512, 513, 1500, 2048, 2049, 9000])
@pytest.mark.parametrize("width", [1e-3, 0.0, 1e-5])
def test_borders_in_a_crowd(gpu, n, width):
    """Borders of top_k and top_p, alone and together, that fall among n ids which share a bin: lists of every size that is
    ranked by a form of its own, and past 2048 the row that one workgroup takes."""
    rng = np.random.default_rng(n)
    v = 20000
    x = crowd(rng, v, n, width)
    w = np.exp(x.astype(np.float64) - x.max())
    high = np.sort(w)[::-1].cumsum()
    total = w.sum()
    p = float((high[6] + 0.41 * (high[5 + n] - high[6])) / total) if n > 1 else 0.9
    k = 6 + max(1, int(0.6 * n))
    sets = [(1.0, k, 1.0, 0.0), (1.0, 0, p, 0.0), (1.0, k, 0.97 * p, 0.0), (1.0, k, 0.7, 0.01), (1.0, 0, p, 0.05), (0.9, 100, 0.95, 0.0), (1.0, 6 + n, 0.99, 0.0),
            (1.0, 20, 1.0, 0.0), (1.0, 128, 0.9, 0.0), (1.0, 1, 1.0, 0.0)]
    check(gpu, np.repeat(x[None], len(sets), 0), sets, rng.random(len(sets)))
    check(gpu, np.repeat(x[None], len(sets), 0), sets, np.full(len(sets), 0.999), probs=False)


@pytest.mark.parametrize("vocab,rows", [(151936, 40), (151935, 130), (5000, 1100), (30, 2500), (1300003, 2), (1100000, 3)])
def test_rounds_and_rows(gpu, vocab, rows):
    """Parts of several rounds (many rows, or a vocabulary past a million ids) and more rows than go at once."""
    rng = np.random.default_rng(rows)
    x = (2 * rng.standard_normal((rows, vocab))).astype(np.float32)
    mix = [(1.0, 40, 0.9, 0.0), (0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.0), (1.0, 500, 0.95, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 0, 1.0, 0.05), (1.2, 128, 1.0, 0.0)]
    sets = [mix[r % len(mix)] for r in range(rows)]
    u = rng.random(rows).astype(np.float32)
    tok, pr = sample(gpu, x, sets, u)
    again, _ = sample(gpu, x, sets, u, probs=False)
    assert np.array_equal(tok, again)
    for r in np.unique(np.concatenate([np.arange(min(rows, 7)), rng.integers(0, rows, 12), [rows - 1, min(1023, rows - 1), min(1024, rows - 1)]])):
        want, probs, margin = P.sample(x[r], *sets[r], u[r])
        assert margin > 1e-11 and int(tok[r].astype(np.int32)) == want
        assert (np.abs(pr[r] - probs) <= probs * (2.0 ** -24 + 1e-9) + 2.0 ** -149).all()
        assert np.array_equal(pr[r] > 0, probs.astype(np.float32) > 0)


@pytest.mark.parametrize("kind", ["sorted", "blocks", "masked", "lowest", "spread"])
def test_logits_in_unkind_orders(gpu, kind):
    """Rows in falling order (all of the largest in one part), equal blocks, few ids allowed, masks of the type's lowest value, and
    logits over a hundred thousand nats."""
    rng = np.random.default_rng(5)
    v = 60000
    x = (3 * rng.standard_normal(v)).astype(np.float32)
    if kind == "sorted":
        x = np.sort(x)[::-1].copy()
    elif kind == "blocks":
        x = np.repeat(x[::600], 600)[:v].copy()
    elif kind == "masked":
        keep = rng.integers(0, v, 90)
        y = np.full(v, -np.inf, np.float32)
        y[keep] = x[keep]
        x = y
    elif kind == "lowest":
        x[rng.random(v) < 0.9] = np.finfo(np.float32).min
    else:
        x = (x * 3e4).astype(np.float32)
    sets = [(1.0, 50, 0.9, 0.0), (1.0, 0, 0.9, 0.0), (1.0, 1000, 0.97, 0.0), (1.0, 1000, 1.0, 0.0), (0.5, 0, 1.0, 0.01), (20.0, 0, 0.6, 0.0), (1.0, 100, 1.0, 0.0),
            (0.0, 5, 0.1, 0.9), (1.0, 0, 1.0, 0.0)]
    check(gpu, np.repeat(x[None], len(sets), 0), sets, rng.random(len(sets)))


def test_infinite_temperature_and_logits(gpu):
    x = np.linspace(-3, 3, 4000).astype(np.float32)
    y = x.copy()
    y[[7, 900, 3999]] = np.inf
    sets = [(np.inf, 0, 1.0, 0.0), (np.inf, 3, 1.0, 0.0), (np.inf, 0, 0.333, 0.0), (1.0, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.5), (np.inf, 2000, 0.9999, 0.1)]
    check(gpu, np.repeat(x[None], len(sets), 0), sets, np.full(len(sets), 0.377))
    check(gpu, np.repeat(y[None], len(sets), 0), sets, np.full(len(sets), 0.377))


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 31, 33, 127, 128, 129, 131, 254, 255, 256, 257, 300])
@pytest.mark.parametrize("width", [1e-3, 0.05, 0.3])
@pytest.mark.parametrize("alike", [False, True])
def test_lists_of_every_short_length(gpu, n, width, alike):
    """Both borders anywhere in a crowd over one bin or several, a quarter of its ids alike or none: the lists that are compared
    all with all, and the first ones past them."""
    rng = np.random.default_rng(n)
    x = crowd(rng, 3000, n, width)
    if alike:
        at = np.flatnonzero(x > 3.9)[::4]
        x[at] = np.float32(4 + width / 2)
    w = np.sort(np.exp(x.astype(np.float64) - x.max()))[::-1].cumsum()
    sets = []
    for a in (0.1, 0.5, 0.93):
        k, p = 6 + max(1, int(a * n)), (w[5] + (a + 0.013) * (w[5 + n] - w[5])) / w[-1]
        sets += [(1.0, k, 1.0, 0.0), (1.0, 0, p, 0.0), (1.0, k, p, 0.0), (1.0, 6 + n, p, 0.0), (1.0, max(k, 140), 0.9 * p, 0.0), (1.0, k, 0.9999, 0.04)]
    check(gpu, np.repeat(x[None], len(sets), 0), sets, rng.random(len(sets)))
    check(gpu, np.repeat(x[None], len(sets), 0), sets, rng.random(len(sets)), probs=False)
