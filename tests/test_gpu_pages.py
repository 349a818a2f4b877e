"""Rows into a paged f16 cache, attention over it and eviction from it, on the
GPU against plain forms in 64 bits (include/surge.h)."""
import ctypes as C
import math

import numpy as np
import pytest

import pages_oracle as P
import surge_amd as S
from test_gpu_kv8 import Bufs
from test_gpu_operator_aliases import Alias

pytestmark = pytest.mark.gpu
F = S.fbits


def b16(a):
    return a.view(np.uint16)


def pools(rng, pages, page, nkv, hd, gain=1.0):
    return [(rng.standard_normal((pages, page, nkv, hd)) * gain).astype(np.float16) for _ in range(2)]


def tables(rng, n, width, free=2):
    """Each sequence its own pages, in no order."""
    pages = n * width + free
    return rng.permutation(pages)[:n * width].reshape(n, width).astype(np.int32), pages


# ---------------------------------------------------------------- store

@pytest.mark.parametrize("nkv,hd,page", [(4, 256, 16), (2, 64, 32), (1, 128, 256), (12, 64, 64), (3, 128, 128), (5, 256, 16)])
@pytest.mark.parametrize("n,rows", [(1, 1), (3, 1), (2, 40), (1, 300), (7, 5)])
@pytest.mark.parametrize("pad", [0, 4, 3])
def test_store(gpu, nkv, hd, page, n, rows, pad):
    rng = np.random.default_rng(nkv * 1000 + rows + pad)
    width = 320 // page + 2
    table, pages = tables(rng, n, width)
    kp, vp = pools(rng, pages, page, nkv, hd)
    cap, w = width * page, nkv * hd
    span = np.stack([[int(rng.integers(0, cap - rows + 1)), rows - (s % 2 if rows > 1 else 0), int(rng.integers(0, 10 ** 6))]
                     for s in range(n)]).astype(np.int32)
    x = [(rng.standard_normal((n, rows, nkv, hd)) * 10.0 ** rng.integers(-6, 4, (n, rows, nkv, 1))).astype(np.float32) for _ in range(2)]
    weight, pos = rng.random((n, nkv, cap)).astype(np.float32), rng.integers(0, 99, (n, nkv, cap)).astype(np.int32)
    stride = w + pad
    flat = []
    for a in x:
        r = np.full((n * rows, stride), np.nan, np.float32)
        r[:, :w] = a.reshape(n * rows, w)
        flat.append(r.reshape(-1)[:(n * rows - 1) * stride + w])
    with Bufs(gpu) as buf:
        b = [buf(a) for a in flat + [kp, vp, table, span, weight, pos]]
        gpu.page_store(*b, [nkv, hd, page, n, width, rows, stride if pad else 0])
        got = [b[i].array.copy() for i in (2, 3, 6, 7)]
        gpu.page_store(*b[:6], None, None, [nkv, hd, page, n, width, rows, stride])      # again, without the two
        assert np.array_equal(b16(b[2].array), b16(got[0])) and np.array_equal(b16(b[3].array), b16(got[1]))
    P.store(x[0], x[1], kp, vp, table, span, weight, pos)
    assert np.array_equal(b16(got[0]), b16(kp)) and np.array_equal(b16(got[1]), b16(vp))
    assert np.array_equal(got[2], weight) and np.array_equal(got[3], pos)


def test_store_leaves_out_what_has_no_place(gpu):
    """Padded sequences, rows past the last slot, page numbers outside the pool, counts past n, the largest numbers."""
    rng = np.random.default_rng(1)
    n, rows, nkv, hd, page, width = 9, 20, 2, 64, 16, 2
    table, pages = tables(rng, n, width)
    big = 2 ** 31 - 1
    table[2, 1], table[3, 0], table[4] = pages, -1, big
    span = np.array([[-1, 20, 0], [5, 0, 0], [10, 20, 7], [10, 20, 9], [0, 20, 0], [25, 20, 3], [12, big, -5], [big, big, big], [3, -4, 0]],
                    np.int32)
    kp, vp = pools(rng, pages, page, nkv, hd)
    k, v = rng.standard_normal((2, n, rows, nkv, hd)).astype(np.float32)
    weight, pos = np.ones((n, nkv, 32), np.float32), np.full((n, nkv, 32), 7, np.int32)
    with Bufs(gpu) as buf:
        b = [buf(a) for a in (k, v, kp, vp, table, span, weight, pos)]
        gpu.page_store(*b, [nkv, hd, page, n, width, rows])
        got = [b[i].array.copy() for i in (2, 3, 6, 7)]
    P.store(k, v, kp, vp, table, span, weight, pos)
    for a, want in zip(got, (kp, vp, weight, pos)):
        assert a.tobytes() == want.tobytes()


def test_store_rounds_as_f16_does(gpu):
    x = np.array([0.0, -0.0, 1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 1 + 2.0 ** -11 + 2.0 ** -20, 65504, 65519.996, 65520, -1e9, np.inf, -np.inf, np.nan,
                  2.0 ** -24, 2.0 ** -25, 1.5 * 2.0 ** -24, 2.0 ** -25 * 1.0001, 2.0 ** -14, 6.1e-5, -3e-8, 1e-40], np.float32)
    row = np.zeros((1, 1, 1, 64), np.float32)
    row[0, 0, 0, :len(x)] = x
    with Bufs(gpu) as buf:
        kp, vp = buf(np.zeros((1, 16, 1, 64), np.float16)), buf(np.zeros((1, 16, 1, 64), np.float16))
        gpu.page_store(buf(row), buf(row), kp, vp, buf(np.zeros((1, 1), np.int32)), buf(np.array([[3, 1, 0]], np.int32)), None, None,
                       [1, 64, 16, 1, 1, 1])
        with np.errstate(over="ignore"):
            want = row[0, 0, 0].astype(np.float16)
        for b in (kp, vp):
            got = b.array[0, 3, 0]
            assert np.array_equal(np.isnan(got), np.isnan(want))
            assert np.array_equal(b16(got)[~np.isnan(want)], b16(want)[~np.isnan(want)])
            assert not b.array[0, 4:].any() and not b.array[0, :3].any()


# ---------------------------------------------------------------- attention

def attn(gpu, q, kp, vp, table, lens, weight=None, weights=False, scale=None, q_pad=0, tail=0):
    n, nh, hd = q.shape
    page, nkv = kp.shape[1:3]
    width = table.shape[1]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    qs = np.full((n, nh, hd + q_pad), np.nan, np.float32)
    qs[:, :, :hd] = q
    with Bufs(gpu) as buf:
        out = buf(np.full(n * nh * hd + tail, 5.0, np.float32))
        wo = buf(np.full((n, nkv, width * page), -3.0, np.float32)) if weights or weight is not None else None
        gpu.attn_paged(buf(qs.reshape(-1)[:(n * nh - 1) * (hd + q_pad) + hd]), buf(kp), buf(vp), buf(table), buf(np.asarray(lens, np.int32)),
                       buf(weight) if weight is not None else None, wo, out,
                       [nh, nkv, hd, page, n, width, hd + q_pad, F(scale)])
        assert (out.array[n * nh * hd:] == 5.0).all()
        return out.array[:n * nh * hd].reshape(n, nh, hd).copy(), wo.array.copy() if wo is not None else None


def check_attn(gpu, q, kp, vp, table, lens, weight=None, weights=False, scale=None, **kw):
    hd = q.shape[2]
    got, wo = attn(gpu, q, kp, vp, table, lens, weight, weights, scale, **kw)
    want, bound, w, wb = P.attn(q, kp, vp, table, lens, np.float32(1 / math.sqrt(hd) if scale is None else scale), weight)
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) / bound).max())
    if wo is not None:
        cap = w.shape[2]
        held = np.arange(cap) < np.clip(np.asarray(lens, np.int64), 0, cap)[:, None, None]
        held = np.broadcast_to(held, w.shape)
        assert (wo[~held] == -3.0).all()
        assert (np.abs(wo - w) <= wb)[held].all()
    return got, wo


SHAPES = [(24, 4, 256, 16), (8, 2, 256, 32), (16, 4, 256, 64), (32, 8, 128, 64), (12, 12, 64, 16), (16, 1, 128, 256), (16, 1, 256, 128),
          (3, 1, 64, 32), (5, 5, 128, 16), (30, 2, 64, 128)]


@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
@pytest.mark.parametrize("lens", [[1], [0, 16, 1, 17], [33, 0, 31, 32, 15, 64, 65], [700], [257, 511, 512, 513, 3], [2300, 5]])
def test_attn(gpu, nh, nkv, hd, page, lens):
    rng = np.random.default_rng(nh + hd + len(lens) + sum(lens))
    n = len(lens)
    table, pages = tables(rng, n, -(-max(max(lens), 1) // page) + 1)
    kp, vp = pools(rng, pages, page, nkv, hd)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    check_attn(gpu, q, kp, vp, table, lens)
    weight = rng.random((n, nkv, table.shape[1] * page)).astype(np.float32)
    check_attn(gpu, q, kp, vp, table, lens, weight, tail=3)
    check_attn(gpu, q, kp, vp, table, lens, weights=True, q_pad=hd)       # query | gate rows
    check_attn(gpu, q, kp, vp, table, lens, q_pad=3)


@pytest.mark.parametrize("nh,nkv,hd,page,lens", [(24, 4, 256, 64, [20011]), (12, 12, 64, 256, [30001, 7]), (16, 1, 128, 16, [9000] * 3)])
def test_attn_long(gpu, nh, nkv, hd, page, lens):
    rng = np.random.default_rng(hd)
    n = len(lens)
    table, pages = tables(rng, n, -(-max(lens) // page))
    kp, vp = pools(rng, pages, page, nkv, hd)
    check_attn(gpu, rng.standard_normal((n, nh, hd)).astype(np.float32), kp, vp, table, lens, weights=True)


def test_attn_many_sequences(gpu):
    rng = np.random.default_rng(12)
    n, nh, nkv, hd, page = 301, 4, 2, 64, 16
    lens = rng.integers(0, 90, n)
    table, pages = tables(rng, n, 6)
    kp, vp = pools(rng, pages, page, nkv, hd)
    check_attn(gpu, rng.standard_normal((n, nh, hd)).astype(np.float32), kp, vp, table, lens, weights=True)


@pytest.mark.parametrize("nh,nkv,hd,page", [(24, 4, 256, 32), (12, 12, 64, 16), (32, 8, 128, 64)])
def test_attn_reads_nothing_behind_a_sequence(gpu, nh, nkv, hd, page):
    """NaN and infinities in every row that no length covers, and in pages that no table names."""
    rng = np.random.default_rng(3)
    lens = [page + 1, 0, 3 * page - 1, 70, 1, 5 * page]
    n = len(lens)
    table, pages = tables(rng, n, 6)
    kp, vp = pools(rng, pages, page, nkv, hd)
    used = np.zeros((pages, page), bool)
    for s in range(n):
        for j in range(lens[s]):
            used[P.where(table, pages, page, s, j)] = True
    for pool, poison in ((kp, [np.nan, np.inf, -np.inf]), (vp, [np.inf, np.nan, -np.inf])):
        pool[~used] = np.array(poison, np.float16)[rng.integers(0, 3, (~used).sum())][:, None, None]
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    clean, _ = check_attn(gpu, q, kp, vp, table, lens, weights=True)
    for s in range(n):          # what stands in the table behind a sequence's pages does not count either
        table[s, -(-lens[s] // page):] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31, 0], 6 - -(-lens[s] // page))
    again, _ = check_attn(gpu, q, kp, vp, table, lens, weights=True)
    assert np.array_equal(clean, again)


def test_attn_passes_over_pages_outside_the_pool(gpu):
    rng = np.random.default_rng(4)
    nh, nkv, hd, page, width = 8, 2, 64, 16, 5
    lens = [80, 41, 80, 16, -7, 10 ** 9, 2 ** 31 - 1, -2 ** 31]
    n = len(lens)
    table, pages = tables(rng, n, width)
    table[0, 2], table[1, 2], table[2], table[3, 0], table[5, 0], table[6, 4] = -1, pages, [-1, 2 ** 31 - 1, -2 ** 31, pages, pages + 1], -9, pages, -1
    kp, vp = pools(rng, pages, page, nkv, hd)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    got, _ = check_attn(gpu, q, kp, vp, table, lens, rng.random((n, nkv, 80)).astype(np.float32))
    for s in (2, 3, 4, 7):
        assert not got[s].any()


def test_attn_of_shared_pages_and_a_plain_cache(gpu):
    """Continuations of one prompt: its pages in every table. And a cache without pages, seen as one."""
    rng = np.random.default_rng(5)
    nh, nkv, hd, page = 24, 4, 256, 64
    table = np.array([[3, 1, 0], [3, 1, 2], [3, 1, 4]], np.int32)
    kp, vp = pools(rng, 5, page, nkv, hd)
    lens = [130, 190, 129]
    q = rng.standard_normal((3, nh, hd)).astype(np.float32)
    check_attn(gpu, q, kp, vp, table, lens, rng.random((3, nkv, 192)).astype(np.float32))
    seq = 300
    got, _ = check_attn(gpu, q[:1], kp, vp, np.arange(5, dtype=np.int32)[None], [seq], weights=True)
    with Bufs(gpu) as buf:
        out = buf(np.zeros((nh, hd), np.float32))
        gpu.attn_decode_f16(buf(q[0]), buf(kp.reshape(-1, nkv, hd)[:seq]), buf(vp.reshape(-1, nkv, hd)[:seq]), out,
                            [nh, nkv, hd, seq, hd, F(1 / math.sqrt(hd))])
        assert np.abs(out.array - got[0]).max() < 1e-3


@pytest.mark.parametrize("gain,scale", [(1.0, 30.0), (200.0, 1.0), (1e-3, 0.1), (1.0, -0.2), (1.0, 0.0), (60000.0, 1e-4)])
@pytest.mark.parametrize("qgain", [1.0, 1e-6, 1e-38, 1e12])
def test_attn_scores_of_every_size(gpu, gain, scale, qgain):
    """Scores from nothing to thousands; q far from one (its scale put back so that scores stay the same)."""
    rng = np.random.default_rng(6)
    nh, nkv, hd, page, lens = 6, 1, 128, 16, [333, 40]
    table, pages = tables(rng, 2, 21)
    kp, vp = pools(rng, pages, page, nkv, hd, 0.3)
    kp = np.clip(kp.astype(np.float64) * gain, -65504, 65504).astype(np.float16)
    q = (rng.standard_normal((2, nh, hd)) * qgain).astype(np.float32)
    scale = np.float32(scale / qgain)
    if not np.isfinite(scale):
        return
    check_attn(gpu, q, kp, vp, table, lens, weights=True, scale=scale)


def test_attn_one_row_takes_all_and_rows_alike(gpu):
    rng = np.random.default_rng(7)
    nh, nkv, hd, page = 4, 2, 64, 16
    table, pages = tables(rng, 2, 40)
    kp, vp = pools(rng, pages, page, nkv, hd)
    q = rng.standard_normal((2, nh, hd)).astype(np.float32)
    a, b = P.where(table, pages, page, 0, 611)
    kp[a, b] = (np.sign(q[0, ::2]) * 3000).astype(np.float16)
    got, _ = check_attn(gpu, q, kp, vp, table, [640, 640], weights=True)
    assert np.array_equal(got[0, ::2], vp[a, b].astype(np.float32))        # one row's value, exactly
    kp[...] = kp[0, 0]
    _, w = check_attn(gpu, q, kp, vp, table, [640, 513], weights=True)
    assert np.allclose(w[1, :, :513], 2 / 513, rtol=1e-5)


def test_attn_of_rows_that_are_not_finite(gpu):
    rng = np.random.default_rng(8)
    nh, nkv, hd, page = 8, 2, 64, 16
    table, pages = tables(rng, 1, 6)
    q = rng.standard_normal((1, nh, hd)).astype(np.float32)
    for bad in (np.nan, np.inf):
        kp, vp = pools(rng, pages, page, nkv, hd)
        a, b = P.where(table, pages, page, 0, 50)
        kp[a, b, 0, 3] = bad
        vp[a, b, 1, 5] = bad
        got, _ = attn(gpu, q, kp, vp, table, [90], weights=True)
        for c in range(4):          # NaN, or where the row's score is -inf what the other rows give
            one = np.concatenate([kp[table[0]].reshape(-1, nkv, hd)[:90, 0], vp[table[0]].reshape(-1, nkv, hd)[:90, 0]], axis=1)
            one = np.delete(one, 50, axis=0).astype(np.float64)
            e = np.exp(one[:, :hd] @ q[0, c] / 8)
            assert np.isnan(got[0, c]).all() or (bad > 0 and q[0, c, 3] < 0 and np.allclose(got[0, c], e @ one[:, hd:] / e.sum(), atol=1e-4))
        assert not np.isfinite(got[0, 4:, 5]).any() and np.isfinite(np.delete(got[0, 4:], 5, axis=1)).all()
        q2 = q.copy()
        kp, vp = pools(rng, pages, page, nkv, hd)
        q2[0, 1, 7] = bad
        got, _ = attn(gpu, q2, kp, vp, table, [90])
        assert np.isnan(got[0, 1]).all() and np.isfinite(np.delete(got[0], 1, axis=0)).all()


def test_attn_again_and_in_place(gpu):
    """The same bits on a second call; weight and weight_out one buffer, by one handle and by two."""
    rng = np.random.default_rng(9)
    nh, nkv, hd, page, lens = 24, 4, 256, 16, [700, 33]
    table, pages = tables(rng, 2, 44)
    kp, vp = pools(rng, pages, page, nkv, hd)
    q = rng.standard_normal((2, nh, hd)).astype(np.float32)
    weight = rng.random((2, nkv, 704)).astype(np.float32)
    first, w = attn(gpu, q, kp, vp, table, lens, weight)
    again, w2 = attn(gpu, q, kp, vp, table, lens, weight)
    assert np.array_equal(first, again) and np.array_equal(w, w2)
    p = [nh, nkv, hd, page, 2, 44, hd, F(1 / math.sqrt(hd))]
    held = np.arange(704) < np.array(lens)[:, None, None]
    want = np.where(held, w, weight)
    with Bufs(gpu) as buf:
        b = [buf(a) for a in (q, kp, vp, table, np.array(lens, np.int32))]
        out, one, two = buf(np.zeros_like(q)), buf(weight), buf(weight)
        gpu.attn_paged(*b, one, one, out, p)
        assert np.array_equal(one.array, want) and np.array_equal(out.array, first)
        a = Alias(gpu, two, two.nbytes)
        gpu.attn_paged(*b, two, a, out, p)
        assert np.array_equal(two.array, want)
        gpu.attn_paged(*b, a, two, out, p)          # the alias's data, on the device, count: the sums go on
        three = two.array.copy()
        a.free()
    _, w3 = attn(gpu, q, kp, vp, table, lens, want.astype(np.float32))
    assert np.array_equal(three[np.broadcast_to(held, three.shape)], w3[np.broadcast_to(held, three.shape)])


# ---------------------------------------------------------------- eviction

def evict(gpu, kp, vp, table, lens, weight, pos, keep, recent, in_place=False):
    page, nkv, hd = kp.shape[1:]
    with Bufs(gpu) as buf:
        b = [buf(a) for a in (kp, vp, table, np.asarray(lens, np.int32), weight, pos)]
        wo, po = (b[4], b[5]) if in_place else (buf(np.full_like(weight, -3.0)), buf(np.full_like(pos, -3)))
        p = [nkv, hd, page, len(table), table.shape[1], keep, recent]
        gpu.page_evict(*b, wo, po, p)
        r = [b[0].array.copy(), b[1].array.copy(), wo.array.copy(), po.array.copy()]
        if not in_place:        # nothing that the call reads has changed: again the same
            gpu.page_evict(*b, wo, po, p)
            for x, y in zip(r, (b[0], b[1], wo, po)):
                assert x.tobytes() == y.array.tobytes()
        return r


def check_evict(gpu, kp, vp, table, lens, weight, pos, keep, recent):
    k, v = kp.copy(), vp.copy()
    wo, po = P.evict(k, v, table, lens, weight, pos, keep, recent)
    cap = weight.shape[2]
    told = np.broadcast_to(np.arange(cap) < np.minimum(np.clip(np.asarray(lens, np.int64), 0, cap), keep)[:, None, None], weight.shape)
    for in_place in (False, True):
        got = evict(gpu, kp, vp, table, lens, weight, pos, keep, recent, in_place)
        assert np.array_equal(b16(got[0]), b16(k)) and np.array_equal(b16(got[1]), b16(v))
        for a, want, before in ((got[2], wo, weight), (got[3], po, pos)):
            assert a[told].tobytes() == want[told].tobytes()
            assert a[~told].tobytes() == (before[~told] if in_place else np.full_like(a[~told], -3)).tobytes()


def marks(rng, n, nkv, cap, ties=True):
    w = np.exp(2 * rng.standard_normal((n, nkv, cap))).astype(np.float32)
    if ties:
        w[rng.random(w.shape) < 0.3] = 0
        w[rng.random(w.shape) < 0.2] = 1.5
    return w, np.cumsum(rng.integers(1, 4, (n, nkv, cap)), axis=2).astype(np.int32)


@pytest.mark.parametrize("nkv,hd,page", [(4, 256, 16), (12, 64, 32), (1, 128, 64), (3, 128, 256)])
@pytest.mark.parametrize("lens,keep,recent", [([17], 16, 4), ([300, 299, 20, 0, 301], 300, 300), ([1500, 40, 1024, 1025], 40, 7),
                                              ([2], 1, 0), ([2], 1, 1), ([600], 599, 0), ([900, 901], 1, 1), ([500], 400, 0)])
def test_evict(gpu, nkv, hd, page, lens, keep, recent):
    rng = np.random.default_rng(nkv + keep)
    n = len(lens)
    table, pages = tables(rng, n, -(-max(lens) // page) + 1)
    kp, vp = pools(rng, pages, page, nkv, hd)
    weight, pos = marks(rng, n, nkv, table.shape[1] * page)
    check_evict(gpu, kp, vp, table, lens, weight, pos, keep, recent)


@pytest.mark.parametrize("length,keep", [(20000, 2500), (20000, 19999), (70000, 65000), (33000, 32768)])
def test_evict_long(gpu, length, keep):
    rng = np.random.default_rng(keep)
    table, pages = tables(rng, 1, -(-length // 64))
    kp, vp = pools(rng, pages, 64, 2, 64)
    weight, pos = marks(rng, 1, 2, table.shape[1] * 64, ties=keep % 2 == 0)
    check_evict(gpu, kp, vp, table, [length], weight, pos, keep, keep // 10)


def test_evict_weights_of_every_kind(gpu):
    """NaN, infinities, both zeros, subnormals, negatives; all alike; all recent; positions in no order, at the ends of the range."""
    rng = np.random.default_rng(2)
    n, nkv, hd, page, width = 6, 2, 64, 16, 8
    table, pages = tables(rng, n, width)
    kp, vp = pools(rng, pages, page, nkv, hd)
    weight, pos = marks(rng, n, nkv, 128)
    odd = np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 3.4e38, -3.4e38, 1.0], np.float32)
    weight[0] = odd[rng.integers(0, len(odd), (nkv, 128))]
    weight[1], pos[1] = 2.0, 5
    weight[2], pos[2] = np.nan, rng.permutation(128)
    pos[3] = rng.choice([-2 ** 31, 2 ** 31 - 1, 0], (nkv, 128))
    pos[4] = rng.permutation(128)
    weight[5] = 0.0
    for keep, recent in ((50, 10), (128, 128), (1, 1), (100, 0), (64, 64)):
        check_evict(gpu, kp, vp, table, [128, 120, 100, 128, 128, 10 ** 9], weight, pos, keep, recent)


def test_evict_with_pages_outside_the_pool(gpu):
    rng = np.random.default_rng(5)
    table, pages = tables(rng, 2, 6)
    table[0, 0], table[0, 5], table[1, 4] = -1, pages, 2 ** 31 - 1
    kp, vp = pools(rng, pages, 16, 2, 64)
    weight, pos = marks(rng, 2, 2, 96)
    check_evict(gpu, kp, vp, table, [96, 96], weight, pos, 40, 8)
    check_evict(gpu, kp, vp, table, [96, -5], weight, pos, 5000, 8)         # keep past every slot: nothing to do


# ---------------------------------------------------------------- together

@pytest.mark.parametrize("nh,nkv,hd,page,keep", [(8, 2, 64, 16, 40), (24, 4, 256, 32, 33)])
def test_a_run_of_steps(gpu, nh, nkv, hd, page, keep):
    """A prompt's rows into the pages, then steps: store, attention with its weights, eviction, a sampled token; buffers stay
    on the device's side between calls as a program keeps them, and a plain program does the same beside it."""
    rng = np.random.default_rng(nh)
    n, width, steps, recent, vocab = 3, 5, 14, 6, 97
    cap = width * page
    table, pages = tables(rng, n, width)
    kp, vp = np.zeros((2, pages, page, nkv, hd), np.float16)
    lens = np.array([keep - 3, 0, 7], np.int32)
    position = lens.astype(np.int64).copy()
    weight, pos = np.zeros((n, nkv, cap), np.float32), np.zeros((n, nkv, cap), np.int32)
    with Bufs(gpu) as buf:
        dev = {x: buf(a) for x, a in dict(kp=kp, vp=vp, table=table, lens=lens, weight=weight, pos=pos).items()}

        def put(rows, counts):
            k, v = rng.standard_normal((2, n, rows, nkv, hd)).astype(np.float32)
            span = np.stack([lens if rows == 1 else np.zeros(n, int), counts, position if rows == 1 else np.zeros(n, int)], 1).astype(np.int32)
            gpu.page_store(buf(k), buf(v), dev["kp"], dev["vp"], dev["table"], buf(span), dev["weight"], dev["pos"],
                           [nkv, hd, page, n, width, rows])
            P.store(k, v, kp, vp, table, span, weight, pos)

        put(keep, lens.copy())
        for step in range(steps):
            put(1, np.ones(n, int))
            lens += 1
            position += 1
            dev["lens"].array[...] = lens
            q, out = rng.standard_normal((n, nh, hd)).astype(np.float32), buf(np.zeros((n, nh, hd), np.float32))
            gpu.attn_paged(buf(q), dev["kp"], dev["vp"], dev["table"], dev["lens"], dev["weight"], dev["weight"], out,
                           [nh, nkv, hd, page, n, width, hd, F(1 / math.sqrt(hd))])
            want, bound, w, wb = P.attn(q, kp, vp, table, lens, np.float32(1 / math.sqrt(hd)), weight)
            assert (np.abs(out.array - want) <= bound).all()
            assert (np.abs(dev["weight"].array - w) <= wb).all()
            weight = dev["weight"].array.copy()             # its bits decide who stays
            gpu.page_evict(dev["kp"], dev["vp"], dev["table"], dev["lens"], dev["weight"], dev["pos"], dev["weight"], dev["pos"],
                           [nkv, hd, page, n, width, keep, recent])
            weight, pos = P.evict(kp, vp, table, lens, weight, pos, keep, recent)
            lens = np.minimum(lens, keep).astype(np.int32)
            assert np.array_equal(b16(dev["kp"].array), b16(kp)) and np.array_equal(b16(dev["vp"].array), b16(vp))
            assert np.array_equal(dev["weight"].array, weight) and np.array_equal(dev["pos"].array, pos)
            logits = (out.array.reshape(n, -1) @ np.random.default_rng(step).standard_normal((nh * hd, vocab))).astype(np.float32)
            u = rng.random(n).astype(np.float32)
            sets = np.zeros((n, 4), np.float32)
            sets[:, 0], sets[:, 2] = [0.0, 0.8, 1.3], 0.9
            sets[:, 1] = np.array([0, 20, 0], np.uint32).view(np.float32)
            tok = buf(np.zeros(n, np.uint32))
            gpu.sample(buf(logits), buf(sets), buf(u), tok, None, [vocab, n])
            for r in range(n):
                t, _, margin = P.sample(logits[r], sets[r, 0], int(sets[r].view(np.uint32)[1]), 0.9, 0.0, u[r])
                assert margin > 1e-9 and int(tok.array[r]) == t
    assert (position > keep).any()
