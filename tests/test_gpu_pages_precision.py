"""How much of q counts in attention over pages (include/surge.h): every bit of elements near their head's largest, 2^-39 of the largest
of the others."""
import numpy as np
import pytest

from test_gpu_pages import attn, tables

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def exact(q, k, v, scale):
    """out and weights of one sequence in 64 bits: q [heads][hd], k and v [slots][kv heads][hd]."""
    g = len(q) // k.shape[1]
    k, v = k.astype(np.float64), v.astype(np.float64)
    out, size, w = [], [], np.zeros((k.shape[1], len(k)))
    for c, row in enumerate(q.astype(np.float64)):
        x = k[:, c // g] @ row * scale
        p = np.exp(x - x.max())
        p /= p.sum()
        out.append(p @ v[:, c // g])
        size.append(p @ np.abs(v[:, c // g]))
        w[c // g] += p
    return np.array(out), np.array(size), w


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 3, 16])
def test_every_bit_of_q_counts(gpu, hd, group):
    """q's elements differ in their last four bits, and a row of K is 2^15 at one dim and -2^15 at another, so that a score is the
    difference of two elements' last bits, times a power of two: all products and sums on the way are multiples of the last bit's
    product and below 2^24 of them, so that the score is exact, whatever is added first. (Without the bits past 22 scores are off by
    up to a quarter, weights by a fifth.)

    Bounds: x - max is exact and at most 3.75; times log2 e it is off by 1.5 x 2^-24 of it, so that its exponential, with its own
    two, is off by 8 x 2^-24; a sum of 8 slots a lane and step, over 2 steps, 4 lanes, 4 waves and at most 8 parts by 32 x 2^-24;
    quotient and factors 4. So 52 x 2^-24 of a head's weight, and 16 more for the sum over 16 heads. Of the values' sum: the same, two
    halves that hold a weight to 2^-22, and 32 products a step, 2 steps, 4 waves and 8 parts."""
    rng = np.random.default_rng(hd + group)
    n, nkv, page, length = 2, 2, 16, 203
    table, pages = tables(rng, n, 13)
    q = (1 + 2.0 ** -12 + rng.integers(0, 16, (n, nkv * group, hd)) * 2.0 ** -23).astype(np.float32)
    kp = np.zeros((pages, page, nkv, hd), np.float16)
    flat = kp.reshape(-1, hd)
    a = rng.integers(0, hd, len(flat))
    b = (a + rng.integers(1, hd, len(flat))) % hd
    flat[np.arange(len(flat)), a], flat[np.arange(len(flat)), b] = 32768, -32768
    vp = rng.standard_normal(kp.shape).astype(np.float16)
    got, w = attn(gpu, q, kp, vp, table, [length] * n, weights=True, scale=32.0)
    for s in range(n):
        k, v = (x[table[s]].reshape(-1, nkv, hd)[:length] for x in (kp, vp))
        out, size, want = exact(q[s], k, v, 32.0)
        assert (np.abs(w[s, :, :length] - want) <= want * 68 * U).all()
        assert (np.abs(got[s] - out) <= size * (52 + 4 + 80) * U).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("power", [0, 8, 14, 20, 26, 34])
def test_an_element_far_above_the_others(gpu, hd, power):
    """One element of each head 2^power times the others' size, at a dim where K is zero: what is left of the others.

    Bounds: with B the sum of |k| |scale| over a row and A that of |q k| |scale|, a score is off by 2^-39 of the largest element times
    B, and by the f32 sum's A (8 sqrt(hd) + 8) 2^-24 (each rounding half a step of the sum so far, taken as independent and at eight
    times their deviation); a weight by the exponential of twice that, and the roundings above."""
    rng = np.random.default_rng(hd + power)
    n, nh, nkv, page, length = 1, 6, 2, 32, 150
    table, pages = tables(rng, n, 5)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    kp, vp = (rng.standard_normal((pages, page, nkv, hd)).astype(np.float16) for _ in range(2))
    at = rng.integers(0, hd, nkv)
    for h in range(nkv):
        q[0, 3 * h:3 * h + 3, at[h]] = np.float32(2.0 ** power * 1.37)
        kp[:, :, h, at[h]] = 0
    scale = np.float32(1 / np.sqrt(hd))
    got, w = attn(gpu, q, kp, vp, table, [length], weights=True, scale=scale)
    k, v = (x[table[0]].reshape(-1, nkv, hd)[:length] for x in (kp, vp))
    out, size, want = exact(q[0], k, v, float(scale))
    worst = np.zeros(nkv)
    for c in range(nh):
        kk = np.abs(k[:, c // 3].astype(np.float64))
        qq = np.abs(q[0, c].astype(np.float64))
        off = (kk.sum(axis=1).max() * qq.max() * 2.0 ** -39 + (kk @ qq).max() * (8 * np.sqrt(hd) + 8) * U) * scale
        e = np.expm1(2 * off) + 64 * U
        worst[c // 3] = max(worst[c // 3], e)
        assert (np.abs(got[0, c] - out[c]) <= size[c] * (e + 80 * U)).all()
    assert (np.abs(w[0, :, :length] - want) <= want * (worst[:, None] + 8 * U)).all()
