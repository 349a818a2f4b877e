"""Sampled tokens and their distributions on the GPU against a plain form in 64
bits or more (include/surge.h)."""
import ctypes as C

import numpy as np
import pytest

import pages_oracle as P
import surge_amd as S
from test_gpu_kv8 import Bufs
from test_gpu_operator_aliases import Alias

pytestmark = pytest.mark.gpu


def settings(rows):
    s = np.zeros((len(rows), 4), np.uint32)
    for i, (t, k, p, m) in enumerate(rows):
        s[i] = [np.float32(t).view(np.uint32), k, np.float32(p).view(np.uint32), np.float32(m).view(np.uint32)]
    return s


def sample(gpu, x, sets, u, probs=True, in_place=False, tail=0):
    rows, vocab = x.shape
    with Bufs(gpu) as buf:
        tok = buf(np.full(rows + tail, 77, np.uint32))
        full = np.concatenate([x.reshape(-1), np.full(tail, 4.0, np.float32)])
        lx = buf(full)
        pr = lx if in_place else buf(np.full(rows * vocab + tail, 4.0, np.float32)) if probs else None
        gpu.sample(lx, buf(settings(sets)), buf(np.asarray(u, np.float32)), tok, pr, [vocab, rows])
        assert (tok.array[rows:] == 77).all() and (pr is None or (pr.array[rows * vocab:] == 4.0).all())
        return tok.array[:rows].copy(), pr.array[:rows * vocab].reshape(rows, vocab).copy() if pr is not None else None


def check(gpu, x, sets, u, **kw):
    """Tokens equal, the same ids with a probability, each within the roundings of its quotient to f32 (2^-24) and of 64-bit
    exponentials and sums, which are far below."""
    tok, pr = sample(gpu, x, sets, u, **kw)
    for r in range(len(x)):
        want, probs, margin = P.sample(x[r], *sets[r], u[r])
        assert margin > 1e-11, "a border too near for this test's own oracle"
        assert int(tok[r].astype(np.int32)) == want, (r, sets[r], u[r])
        if pr is not None:
            assert np.array_equal(pr[r] > 0, probs.astype(np.float32) > 0)
            assert (np.abs(pr[r] - probs) <= probs * (2.0 ** -24 + 1e-9) + 2.0 ** -149).all()
            assert want < 0 or pr[r, want] > 0
    return tok, pr


MIX = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.8, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 0.95, 0.0), (0.8, 50, 1.0, 0.05), (1.0, 1, 0.3, 0.5),
       (0.6, 0, 0.5, 0.1), (2.0, 1000, 0.99, 0.001), (1.0, 64, 0.9, 0.02), (0.05, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.2), (1.5, 5, 0.7, 0.0)]


def rows_of(rng, rows, vocab, coarse=False):
    x = (3 * rng.standard_normal((rows, vocab))).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, vocab, min(vocab, 5))] += 6
    if coarse:          # many logits alike
        x = (x.view(np.uint32) & np.uint32(0xFFFF0000)).view(np.float32)
    return x


@pytest.mark.parametrize("vocab", [1, 2, 31, 100, 1023, 1024, 1025, 4099, 32000, 151936])
@pytest.mark.parametrize("coarse", [False, True])
def test_sample(gpu, vocab, coarse):
    rng = np.random.default_rng(vocab + coarse)
    x = rows_of(rng, len(MIX), vocab, coarse)
    check(gpu, x, MIX, rng.random(len(MIX)), tail=3)
    a, _ = sample(gpu, x, MIX, [0.5] * len(MIX), probs=False)
    b, p = check(gpu, x, MIX, np.full(len(MIX), 0.5))
    c, q = sample(gpu, x, MIX, [0.5] * len(MIX), in_place=True)
    assert np.array_equal(a, b) and np.array_equal(a, c) and np.array_equal(p, q)


@pytest.mark.parametrize("rows,vocab", [(1, 151936), (3, 151935), (40, 5000), (300, 777), (2, 600001)])
def test_sample_rows(gpu, rows, vocab):
    rng = np.random.default_rng(rows)
    x = rows_of(rng, rows, vocab)
    check(gpu, x, [MIX[(r + rows) % len(MIX)] for r in range(rows)], rng.random(rows))


def test_sample_top_k_and_top_p_over_their_range(gpu):
    """Every top-k up to more ids than there are, and nuclei from the first id to all, over 3000 ids some of them alike."""
    rng = np.random.default_rng(8)
    x = rows_of(rng, 1, 3001, True)
    ks = [1, 2, 3, 7, 8, 9, 63, 64, 65, 255, 256, 257, 1000, 1023, 1024, 1025, 2999, 3000, 3001, 3002, 2 ** 31, 2 ** 32 - 1]
    check(gpu, np.repeat(x, len(ks), 0), [(1.7, k, 1.0, 0.0) for k in ks], rng.random(len(ks)))
    check(gpu, np.repeat(x, len(ks), 0), [(1.7, k, 0.77, 0.0) for k in ks], rng.random(len(ks)))
    ps = [0.0, -1.0, 1e-30, 0.01, 0.1, 0.2, 0.3, 0.4, 0.5, 0.6, 0.7, 0.8, 0.9, 0.97, 0.99, 0.999, 0.99999, 1 - 2.0 ** -24, 1.0, 2.0, np.inf, np.nan]
    for t in (0.9, 30.0):
        check(gpu, np.repeat(x, len(ps), 0), [(t, 0, p, 0.0) for p in ps], rng.random(len(ps)))
    ms = [0.0, -2.0, 1e-6, 1e-3, 0.01, 0.1, 0.35, 0.6, 0.9999, 1.0, 1.5, np.inf, np.nan]
    check(gpu, np.repeat(x, len(ms), 0), [(3.0, 0, 1.0, m) for m in ms], rng.random(len(ms)))


@pytest.mark.parametrize("n", [5, 2000, 40000])
def test_sample_ids_alike(gpu, n):
    """All logits the same: weights of exactly one, borders that fall on ids exactly."""
    x = np.full((6, n), -2.5, np.float32)
    x[1, ::2], x[1, 1::2] = 0.0, -0.0
    sets = [(1.0, 0, 0.5, 0.0), (1.0, 0, 1.0, 1.0), (0.3, n // 2, 1.0, 0.0), (1.0, n // 2, 0.5, 0.0), (0.0, 0, 1.0, 0.0), (2.0, 0, 0.25, 0.9)]
    kept = [-(-n // 2), n, n // 2, -(-(n // 2) // 2), 1, -(-n // 4)]
    u = np.full(6, 0.75, np.float32)
    tok, pr = sample(gpu, x, sets, u)
    for r in range(6):
        assert np.array_equal(np.flatnonzero(pr[r]), np.arange(kept[r]))
        assert (pr[r, :kept[r]] == np.float32(1 / kept[r])).all()
        assert tok[r] == int(0.75 * kept[r])        # the first id i with i + 1 > 0.75 kept


def test_sample_values_that_are_not_finite(gpu):
    rng = np.random.default_rng(3)
    v = 701
    x = rows_of(rng, 8, v)
    x[0, rng.integers(0, v, 400)] = np.nan
    x[1, rng.integers(0, v, 690)] = -np.inf
    x[2] = -np.inf
    x[3] = np.nan
    x[4, [5, 99, 650]] = np.inf
    x[5] = -np.inf
    x[5, 123] = -1e38
    x[6] = np.where(np.arange(v) % 2, -3.4e38, 3.4e38)       # 351 of the largest: no border falls on an id
    x[7] = np.where(np.arange(v) % 3, -np.inf, np.nan)
    for s in MIX:
        tok, _ = check(gpu, x, [s] * 8, rng.random(8))
        assert tok[2] == tok[3] == tok[7] == 0xFFFFFFFF and tok[5] == 123


def test_sample_settings_at_their_ends(gpu):
    rng = np.random.default_rng(4)
    x = rows_of(rng, 1, 5000)
    big = [(np.inf, 0, 1.0, 0.0), (np.inf, 30, 0.49, 0.0), (1e-45, 0, 0.9, 0.0), (1e-30, 10, 1.0, 0.0), (-1.0, 0, 0.5, 0.0), (np.nan, 7, 1.0, 0.0),
           (1e30, 0, 0.37, 0.0), (3.4e38, 0, 1.0, 0.5), (-np.inf, 0, 1.0, 0.0), (1.0, 0, np.nan, np.nan)]
    check(gpu, np.repeat(x, len(big), 0), big, rng.random(len(big)))


def test_sample_random_numbers_at_their_ends(gpu):
    rng = np.random.default_rng(5)
    us = [0.0, -0.0, 1e-45, 1e-9, 2.0 ** -24, 0.5, 1 - 2.0 ** -24, 1.0, 7.0, np.inf, -3.0, -np.inf, np.nan]
    x = rows_of(rng, 1, 2000)
    for s in ((1.0, 0, 1.0, 0.0), (0.8, 40, 0.9, 0.0), (0.4, 0, 1.0, 0.001)):
        tok, _ = sample(gpu, np.repeat(x, len(us), 0), [s] * len(us), us)
        for r, u in enumerate(us):
            assert int(tok[r]) == P.sample(x[0], *s, u)[0], (s, u)
    x[0, :1000] = -np.inf
    x[0, 1999] = -1000.0
    tok, _ = sample(gpu, np.repeat(x, 2, 0), [(1.0, 0, 1.0, 0.0), (1e-3, 0, 1.0, 0.0)], [0.0, 0.0])
    assert tok[0] == 1000 and int(tok[1]) == P.sample(x[0], 1e-3, 0, 1.0, 0.0, 0.0)[0]


def test_sample_frequencies(gpu):
    """Evenly spaced numbers choose each id as often as its probability says, to one."""
    rng = np.random.default_rng(6)
    rows, v = 2000, 300
    x = np.repeat(rows_of(rng, 1, v), rows, 0)
    s = (1.1, 40, 0.93, 0.01)
    tok, _ = sample(gpu, x, [s] * rows, (np.arange(rows) + 0.5) / rows, probs=False)
    _, p, _ = P.sample(x[0], *s, 0.5)
    assert (np.abs(np.bincount(tok, minlength=v) - p * rows) <= 1.0 + 1e-6).all()


def test_sample_in_place_by_two_handles(gpu):
    rng = np.random.default_rng(7)
    x, u = rows_of(rng, 3, 4000), np.array([0.1, 0.6, 0.9], np.float32)
    want, p = check(gpu, x, MIX[1:4], u)
    with Bufs(gpu) as buf:
        src, tok = buf(x), buf(np.zeros(3, np.uint32))
        a = Alias(gpu, src, src.nbytes)
        gpu.sample(src, buf(settings(MIX[1:4])), buf(u), tok, a, [4000, 3])
        assert np.array_equal(tok.array, want) and np.array_equal(src.array, p)
        a.free()
