"""What the attention over the 8-bit cache loses, by each output's own size: blocks
of values whose scales are far apart, against the same in 64 bits."""
import math

import numpy as np
import pytest

import kv8_oracle as K
from test_gpu_kv8 import attend

pytestmark = pytest.mark.gpu


def plain(q, c, base, scale):
    """K.attention's outputs, all rows of a head at once, and the rms error of a score: q's elements to a unit of
    max|q| / (127 2^16), so off by that over sqrt(12) each, and two roundings of its own size (its integers joined,
    its factor), at most u and so u / sqrt(3)."""
    n, nh, hd = q.shape
    g = nh // c.nkv
    k, v = c.values(0, base + n), c.values(1, base + n)
    hide = np.arange(base + n) > np.arange(base, base + n)[:, None]
    out, ds = np.zeros(q.shape), np.zeros((n, nh))
    for h in range(nh):
        s = q[:, h].astype(np.float64) @ k[:, h // g].T * scale
        unit = abs(scale) * np.abs(q[:, h]).max(axis=1) / (127 * 2 ** 16) * np.linalg.norm(k[:, h // g], axis=1).max()
        ds[:, h] = np.sqrt(unit ** 2 / 12 + 2 / 3 * (2.0 ** -24 * np.abs(s).max(axis=1)) ** 2)
        s[hide] = -np.inf
        p = np.exp(s - s.max(axis=1, keepdims=True))
        out[:, h] = p @ v[:, h // g] / p.sum(axis=1, keepdims=True)
    return out, ds


@pytest.mark.parametrize("nh,nkv,hd,block,base,n", [(64, 64, 64, 32, 255, 1), (32, 32, 128, 16, 255, 1), (32, 16, 256, 64, 511, 1),
                                                    (64, 16, 64, 32, 200, 56), (32, 8, 256, 64, 0, 1024), (48, 8, 128, 16, 0, 1024)])
@pytest.mark.parametrize("apart", [2.0 ** -8, 2.0 ** -30, 2.0 ** -60])
@pytest.mark.parametrize("size", [0.0, 0.01, 1.0])
def test_scales_of_any_mantissa_far_apart(gpu, nh, nkv, hd, block, base, n, apart, size):
    """Every second block's values are `apart` times the others', with two scales of a kv head and no power of two
    among them: the small ones count in the sum below alone, and a rounding that all their weights have in common
    does not drop out. In units of u = 2^-24 and as root mean squares, with m keys: a weight 1.4 (exp 2 at most, its
    argument and the two halves), m / 16 additions of a third's root each, the sum below 1 (exp), the small blocks'
    arguments there, up to log2(apart) = 60, half a step of which is 32 ln 2 = 22, over half the keys and weighed by
    a half, the last steps 0.7. A score's error counts in both sums. Three times their root sum of squares."""
    rng = np.random.default_rng(nh + n)
    m = base + n
    c = K.Cache(nkv, hd, block, m)
    c.codes[...] = rng.integers(-127, 128, c.codes.shape)
    c.scales[:, :, 0] = 1 / 60
    c.scales[:, :, 1] = rng.uniform(0.01, 0.02, nkv)
    c.scales[1::2, :, 1] = rng.uniform(1, 2, nkv) * 0.01 * apart
    q = (rng.standard_normal((n, nh, hd)) * size).astype(np.float32)
    want, ds = plain(q, c, base, 1 / math.sqrt(hd))
    got = attend(gpu, c, q, base, 1 / math.sqrt(hd), "decode" if n == 1 else "prefill").astype(np.float64)
    keys = np.arange(base + 1, m + 1)
    u = 2.0 ** -24
    rest = 1.4 ** 2 + keys / 48 + 1 + 0.25 * (22 / math.sqrt(3)) ** 2 / np.maximum(keys / 2, 1) + 0.7 ** 2
    tol = 3 * np.sqrt(u ** 2 * rest[:, None] + (2 * ds) ** 2)
    err = np.linalg.norm(got - want, axis=2) / np.linalg.norm(want, axis=2) / tol
    seen = keys > 2 * block          # both kinds
    assert (err[seen] <= 1).all(), f"worst error {err[seen].max():.2f} of its tolerance, which is {tol[-1].mean() / u:.1f} u"


FORMS = [(8, 2, 128, 32, 99, 1), (24, 4, 256, 64, 2999, 1), (12, 12, 64, 16, 200, 20), (32, 8, 256, 64, 0, 1024), (12, 12, 64, 32, 0, 2500)]


@pytest.mark.parametrize("nh,nkv,hd,block,base,n", FORMS)
def test_one_key_has_all_the_weight(gpu, nh, nkv, hd, block, base, n):
    """Rows whose best key is exp(40) ahead are its values, with a weight's two halves between (2^-22, 4 u), the
    sum of their products 2 and the division 1.5: to 8 u of every element."""
    rng = np.random.default_rng(n)
    m = base + n
    c = K.Cache(nkv, hd, block, m)
    c.codes[...] = rng.integers(-127, 128, c.codes.shape)
    c.scales[...] = rng.uniform(0.01, 0.02, c.scales.shape)
    q = (rng.standard_normal((n, nh, hd)) * 1e3).astype(np.float32)
    got = attend(gpu, c, q, base, 1 / math.sqrt(hd), "decode" if n == 1 else "prefill")
    k, v = c.values(0, m), c.values(1, m)
    hide = np.arange(m) > np.arange(base, m)[:, None]
    checked = 0
    for h in range(nh):
        s = q[:, h].astype(np.float64) @ k[:, h * nkv // nh].T / math.sqrt(hd)
        s[hide] = -np.inf
        best = s.argmax(axis=1)
        top = s[np.arange(n), best]
        s[np.arange(n), best] = -np.inf
        clear = top - s.max(axis=1) > 41
        want = v[best, h * nkv // nh]
        assert (np.abs(got[:, h] - want)[clear] <= 8 * 2.0 ** -24 * np.abs(want)[clear] + 1e-12).all()
        checked += clear.sum()
    assert checked >= n * nh / 2


@pytest.mark.parametrize("nh,nkv,hd,block,base,n", FORMS)
@pytest.mark.parametrize("rise", [0.1, 0.6, 1.5, 2.6, 30.0, -0.7])
def test_scores_that_rise_with_the_keys(gpu, nh, nkv, hd, block, base, n, rise):
    """A block of 16 keys is `rise` ahead of the one before it, in the exponents of two: maxima that pass the one kept
    a little, by little steps, by large ones, and never. Tolerance as above, without the small blocks."""
    rng = np.random.default_rng(n)
    m = base + n
    c = K.Cache(nkv, hd, 16, m)
    c.codes[...] = rng.integers(-127, 128, c.codes.shape)
    c.codes[:, :, 0] = rng.integers(50, 100, c.codes[:, :, 0].shape)
    q = rng.uniform(0.5, 1.5, (n, nh, hd)).astype(np.float32)
    scale = 1 / math.sqrt(hd)
    c.scales[:, :, 0] = np.arange(1, len(c.scales) + 1)[:, None] * (abs(rise) * math.log(2) / (75 * hd * scale))
    c.scales[:, :, 1] = rng.uniform(0.01, 0.02, (len(c.scales), nkv))
    q *= np.float32(math.copysign(1, rise))
    want, ds = plain(q, c, base, scale)
    got = attend(gpu, c, q, base, scale, "decode" if n == 1 else "prefill").astype(np.float64)
    keys, u = np.arange(base + 1, m + 1), 2.0 ** -24
    tol = 3 * np.sqrt(u ** 2 * (1.4 ** 2 + keys / 48 + 1 + 0.7 ** 2)[:, None] + (2 * ds) ** 2)
    err = np.linalg.norm(got - want, axis=2) / np.linalg.norm(want, axis=2) / tol
    assert (err <= 1).all(), f"worst error {err.max():.2f} of its tolerance"


@pytest.mark.parametrize("nh,nkv,hd,block,base,n", FORMS)
@pytest.mark.parametrize("size", [1e5, 1e6, 1e7, 1e8, 1e15, 1e30])
def test_scores_far_from_zero(gpu, nh, nkv, hd, block, base, n, size):
    """Scores past 2^20, and past 2^24, where their steps are larger than one: every second head's q times `size`.
    Such a row is all its best key's (rows whose next one is within the scores' rounding are left out; 8 u as above),
    and the rows beside it, in the same waves, are what they are by themselves."""
    rng = np.random.default_rng(n)
    m = base + n
    c = K.Cache(nkv, hd, block, m)
    c.codes[...] = rng.integers(-127, 128, c.codes.shape)
    c.scales[...] = rng.uniform(0.01, 0.02, c.scales.shape)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    small, scale, u = q.copy(), 1 / math.sqrt(hd), 2.0 ** -24
    q[:, ::2] *= np.float32(size)
    entry = "decode" if n == 1 else "prefill"
    got = attend(gpu, c, q, base, scale, entry)
    assert np.isfinite(got).all()
    want, ds = plain(small, c, base, scale)
    keys = np.arange(base + 1, m + 1)
    tol = 3 * np.sqrt(u ** 2 * (1.4 ** 2 + keys / 48 + 1 + 0.7 ** 2)[:, None] + (2 * ds) ** 2)
    err = np.linalg.norm(got - want, axis=2) / np.linalg.norm(want, axis=2) / tol
    assert (err[:, 1::2] <= 1).all()
    k, v = c.values(0, m), c.values(1, m)
    hide = np.arange(m) >= keys[:, None]
    checked = 0
    for h in range(0, nh, 2):
        s = q[:, h].astype(np.float64) @ k[:, h * nkv // nh].T * scale
        s[hide] = -np.inf
        best = s.argmax(axis=1)
        top = s[np.arange(n), best]
        s[np.arange(n), best] = -np.inf
        # a score's rounding: a unit of q's in every dim, and 16 of its own size
        off = scale * 2 * u * np.abs(q[:, h]).max(axis=1) * np.abs(k[:, h * nkv // nh]).sum(axis=1).max() + 16 * u * np.abs(top)
        clear = top - s.max(axis=1) > 2 * off + 41
        one = v[best, h * nkv // nh]
        assert (np.abs(got[:, h] - one)[clear] <= 8 * u * np.abs(one)[clear] + 1e-12).all()
        checked += clear.sum()
    assert checked >= n * nh / 4


@pytest.mark.parametrize("nh,nkv,hd,block,base,n", FORMS)
@pytest.mark.parametrize("far", [-3e7, -1e10, 3e7, 1e10])
def test_all_scores_far_from_zero(gpu, nh, nkv, hd, block, base, n, far):
    """Every key alike, its score `far` from zero on either side: the mean of the values."""
    rng = np.random.default_rng(n)
    m = base + n
    c = K.Cache(nkv, hd, block, m)
    c.codes[...] = rng.integers(-127, 128, c.codes.shape)
    c.codes[:, :, 0] = 100
    c.scales[:, :, 0] = 0.01
    c.scales[:, :, 1] = rng.uniform(0.01, 0.02, c.scales.shape[:2])
    q = np.full((n, nh, hd), far / math.sqrt(hd), np.float32)
    got = attend(gpu, c, q, base, 1 / math.sqrt(hd), "decode" if n == 1 else "prefill")
    want, _ = plain(q * 0, c, base, 1.0)
    keys, u = np.arange(base + 1, m + 1), 2.0 ** -24
    tol = 3 * u * np.sqrt(1.4 ** 2 + keys / 48 + 1 + 0.7 ** 2)
    assert np.isfinite(got).all()
    assert (np.linalg.norm(got - want, axis=2) / np.linalg.norm(want, axis=2) <= tol[:, None]).all()
