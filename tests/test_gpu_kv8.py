"""The 8-bit K/V cache on the GPU: store and load bit for bit against the exact
quantiser, decode and chunk attention against plain attention in 64 bits over
the values the cache stands for (include/surge.h)."""
import ctypes as C
import math

import numpy as np
import pytest

import kv8_oracle as K
import surge_amd as S

pytestmark = pytest.mark.gpu
F = S.fbits


class Bufs:
    """Buffers of one test, freed at its end."""

    def __init__(self, gpu):
        self.gpu, self.all = gpu, []

    def __call__(self, x):
        b = self.gpu.buf(x)
        self.all.append(b)
        return b

    def __enter__(self):
        return self

    def __exit__(self, *a):
        for b in self.all:
            b.free()


def store(gpu, c, k, v, base, stride=0):
    """The library's store into the oracle cache's arrays (codes, scales afterwards)."""
    with Bufs(gpu) as buf:
        codes, scales = buf(c.codes), buf(c.scales)
        if stride:
            n, w = len(k), c.nkv * c.hd
            rows = []
            for x in (k, v):
                r = np.full((n, stride), np.nan, np.float32)        # gaps must not be read
                r[:, :w] = x.reshape(n, w)
                rows.append(buf(r.reshape(-1)[:(n - 1) * stride + w]))
        else:
            rows = [buf(k), buf(v)]
        gpu.kv8_store(rows[0], rows[1], codes, scales, [c.nkv, c.hd, c.block, base, len(k), stride])
        return codes.array.copy(), scales.array.copy()


def rows(rng, n, nkv, hd, gain=1.0):
    return (rng.standard_normal((2, n, nkv, hd)) * gain).astype(np.float32)


def same(c, got):
    assert np.array_equal(got[1].view(np.uint32), c.scales.view(np.uint32))
    assert np.array_equal(got[0], c.codes)


SHAPES = [(1, 64, 16), (2, 64, 128), (3, 128, 32), (2, 256, 16), (4, 256, 64), (1, 256, 128), (12, 64, 32)]


@pytest.mark.parametrize("nkv,hd,block", SHAPES)
@pytest.mark.parametrize("base,n", [(0, 1), (0, 16), (5, 1), (15, 2), (0, 33), (31, 97), (77, 51), (128, 64), (63, 1)])
def test_store_bits(gpu, nkv, hd, block, base, n):
    rng = np.random.default_rng(base * 100 + n)
    c = K.Cache(nkv, hd, block, base + n + 20, rng)         # with what an earlier sequence left
    old = rows(rng, base, nkv, hd)
    if base:
        c.store(old[0], old[1], 0)
    k, v = rows(rng, n, nkv, hd, 3.0 if n % 2 else 0.5)     # scales that grow, and that do not
    want = c
    before = c.codes.copy(), c.scales.copy()
    got_c = K.Cache(nkv, hd, block, base + n + 20)
    got_c.codes, got_c.scales = before
    got = store(gpu, got_c, k, v, base)
    want.store(k, v, base)
    same(want, got)


def test_store_row_stride_and_alignment(gpu):
    rng = np.random.default_rng(1)
    for stride in (384, 385, 2 * 192):
        c, d = K.Cache(3, 64, 32, 50), K.Cache(3, 64, 32, 50)
        k, v = rows(rng, 40, 3, 64)
        c.store(k, v, 7)
        same(c, store(gpu, d, k, v, 7, stride))


def test_store_one_by_one(gpu):
    """A decode's way of filling blocks: every step against the oracle's own state."""
    rng = np.random.default_rng(2)
    c = K.Cache(2, 128, 32, 48)
    with Bufs(gpu) as buf:
        codes, scales = buf(c.codes), buf(c.scales)
        for i in range(40):
            k, v = rows(rng, 1, 2, 128, 0.3 + 0.1 * i)
            c.store(k, v, i)
            gpu.kv8_store(buf(k), buf(v), codes, scales, [2, 128, 32, i, 1])
            assert np.array_equal(codes.array, c.codes) and np.array_equal(scales.array, c.scales), i


def test_store_special_values(gpu):
    """Ties at half steps, zeros, values near f32's smallest and f16's largest; a value f16 cannot
    hold poisons its block and head only, until the block is stored from its start."""
    c, d = K.Cache(2, 64, 16, 160), K.Cache(2, 64, 16, 160)
    x = np.zeros((160, 2, 64), np.float32)
    tiny = np.float32(1.4e-45)                              # 2^-149
    x[96:112, 0] = (np.arange(64) * 3) * tiny               # 189 steps: a scale of one step, values of 190 of it
    x[96:112, 1] = -(np.arange(64) + 2) * 2 * tiny
    x[112:128, 0] = np.arange(64) * np.float32(1e-41)
    x[112:128, 1] = np.random.default_rng(4).standard_normal((16, 64)) * 1e-37
    x[128:144] = np.random.default_rng(5).standard_normal((16, 2, 64)) * 1e-20
    x[0:16, :, 0] = 127.0                                   # a scale of one
    x[0:16, :, 1:32] = np.arange(31) + 0.5                  # ties
    x[0:16, :, 32:] = np.nextafter(np.arange(32, dtype=np.float32) + 0.5, np.float32(0))
    x[16:32, 0] = 1e-44                                     # a scale that is a few of the smallest steps
    x[16:32, 1, ::3] = -3e-45
    x[32:48, 0, 5], x[32:48, 1, 5] = 65519.0, -65519.0
    x[48:64, 0] = np.random.default_rng(3).standard_normal((16, 64))
    x[50, 0, 3] = np.nan
    x[70, 1, 9] = 65520.0
    x[85, 0, 0] = -np.inf
    c.store(x, -x, 0)
    got = store(gpu, d, x, -x, 0)
    assert np.isnan(c.scales).any() and np.array_equal(np.isnan(got[1]), np.isnan(c.scales))
    ok = ~np.isnan(c.scales)
    assert np.array_equal(got[1][ok], c.scales[ok]) and np.array_equal(got[0], c.codes)
    d.codes, d.scales = got
    # the poisoned block goes on poisoned, and is whole again from its start
    y = np.ones((2, 2, 64), np.float32)
    more = store(gpu, d, y, y, 90)
    assert np.isnan(more[1][5, 0]).all() and not np.isnan(more[1][5, 1]).any()
    d.codes, d.scales = more
    again = store(gpu, d, y, y, 80)
    assert (again[1][5] == np.float32(1) / np.float32(127)).all()


@pytest.mark.parametrize("nkv,hd,block", SHAPES)
@pytest.mark.parametrize("base,n", [(0, 1), (0, 48), (13, 38), (63, 2)])
def test_load_bits(gpu, nkv, hd, block, base, n):
    rng = np.random.default_rng(n)
    c = K.Cache(nkv, hd, block, base + n + 3, rng)
    want = [(c.rows(h, base, base + n).astype(np.float32) *
             c.scales[np.arange(base, base + n) // block, :, h][:, :, None]) for h in range(2)]
    w = nkv * hd
    for stride in (0, w + 1, w + 4):
        st = stride or w
        with Bufs(gpu) as buf:
            mark = np.full((n - 1) * st + w, 7.0, np.float32)
            k, v = buf(mark), buf(mark)
            gpu.kv8_load(buf(c.codes), buf(c.scales), k, v, [nkv, hd, block, base, n, stride])
            for got, x in zip((k.array, v.array), want):
                full = np.full(n * st, 7.0, np.float32)
                full.reshape(n, st)[:, :w] = x.reshape(n, w)
                assert np.array_equal(got, full[:len(got)])


def attend(gpu, c, q, base, scale, entry="prefill", q_stride=0):
    n, nh, hd = q.shape
    qs = q_stride or hd
    qr = np.full((n, nh, qs), np.nan, np.float32)           # gaps must not be read
    qr[:, :, :hd] = q
    with Bufs(gpu) as buf:
        out = buf(np.full((n, nh, hd), np.nan, np.float32))
        if entry == "decode":
            gpu.attn_decode_kv8(buf(qr), buf(c.codes), buf(c.scales), out, [nh, c.nkv, hd, base + 1, qs, F(scale), c.block])
        else:
            gpu.attn_prefill_kv8(buf(qr), buf(c.codes), buf(c.scales), out, [nh, c.nkv, hd, base, n, qs, F(scale), c.block])
        return out.array.copy()


def filled(rng, nkv, hd, block, n, room=40):
    """A cache of n positions; behind them garbage, and NaN scales in blocks wholly behind."""
    c = K.Cache(nkv, hd, block, n + room, rng)
    k = rng.integers(-127, 128, c.codes.shape).astype(np.int8)
    c.codes[...] = k
    c.scales[...] = (np.abs(rng.standard_normal(c.scales.shape)) + 0.3).astype(np.float32) / 60
    c.scales[-(-n // block):] = np.nan
    return c


def close(got, want, bound):
    err = np.abs(got.astype(np.float64) - want)
    assert np.isfinite(got).all()
    assert (err <= bound).all(), f"worst error {float((err / bound).max()):.3f} of its bound"


GROUPS = [(1, 1, 64), (6, 1, 256), (24, 4, 256), (8, 2, 128), (16, 1, 64), (12, 12, 64), (14, 2, 256), (16, 16, 128)]


@pytest.mark.parametrize("nh,nkv,hd", GROUPS)
@pytest.mark.parametrize("seq,block", [(1, 16), (2, 64), (15, 16), (16, 32), (17, 16), (31, 128), (32, 16), (33, 32), (64, 64),
                                       (65, 16), (127, 32), (129, 128), (513, 16), (1000, 64)])
def test_decode(gpu, nh, nkv, hd, seq, block):
    rng = np.random.default_rng(seq * 7 + nh)
    c = filled(rng, nkv, hd, block, seq)
    q = rng.standard_normal((1, nh, hd)).astype(np.float32)
    want, bound = K.attention(q, c, seq - 1, 1 / math.sqrt(hd))
    close(attend(gpu, c, q, seq - 1, 1 / math.sqrt(hd), "decode"), want, bound)


@pytest.mark.parametrize("nh,nkv,hd,seq,block", [(24, 4, 256, 9001, 64), (8, 2, 256, 20011, 16), (3, 1, 64, 33333, 32)])
def test_decode_long(gpu, nh, nkv, hd, seq, block):
    rng = np.random.default_rng(seq)
    c = filled(rng, nkv, hd, block, seq)
    q = rng.standard_normal((1, nh, hd)).astype(np.float32)
    want, bound = K.attention(q, c, seq - 1, 1 / math.sqrt(hd))
    got = attend(gpu, c, q, seq - 1, 1 / math.sqrt(hd), "decode")
    close(got, want, bound)
    assert np.array_equal(got, attend(gpu, c, q, seq - 1, 1 / math.sqrt(hd), "decode"))


@pytest.mark.parametrize("nh,nkv,hd,block,base,n", [
    (24, 4, 256, 64, 17003, 1), (32, 8, 128, 16, 9003, 1), (12, 12, 64, 32, 11999, 1), (24, 4, 256, 32, 11990, 5),
    (16, 8, 128, 128, 9000, 9), (64, 64, 64, 64, 2100, 3)])
def test_few_rows_deep(gpu, nh, nkv, hd, block, base, n):
    """Workgroups of eight waves, whose waves take several steps each."""
    rng = np.random.default_rng(base)
    c = filled(rng, nkv, hd, block, base + n)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    want, bound = K.attention(q, c, base, 1 / math.sqrt(hd))
    got = attend(gpu, c, q, base, 1 / math.sqrt(hd), "decode" if n == 1 else "prefill")
    close(got, want, bound)
    assert np.array_equal(got, attend(gpu, c, q, base, 1 / math.sqrt(hd), "decode" if n == 1 else "prefill"))


@pytest.mark.parametrize("nh,nkv,hd,block,base,n", [(32, 8, 128, 64, 8000, 40), (12, 12, 64, 32, 12001, 60), (16, 16, 128, 16, 33003, 1)])
def test_few_rows_much_work(gpu, nh, nkv, hd, block, base, n):
    """More than 64 steps of 32 keys to a CU: eight waves a workgroup, several steps each, parts joined."""
    rng = np.random.default_rng(base)
    c = filled(rng, nkv, hd, block, base + n)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    want, bound = K.attention(q, c, base, 1 / math.sqrt(hd))
    got = attend(gpu, c, q, base, 1 / math.sqrt(hd))
    close(got, want, bound)
    assert np.array_equal(got, attend(gpu, c, q, base, 1 / math.sqrt(hd)))


@pytest.mark.parametrize("nh,nkv,hd,block", [(8, 2, 256, 32), (6, 1, 64, 16), (16, 1, 128, 64), (4, 4, 128, 128), (10, 2, 64, 32)])
@pytest.mark.parametrize("base,n", [(0, 1), (0, 2), (0, 17), (3, 5), (31, 33), (64, 64), (100, 77), (257, 130), (1000, 3)])
def test_prefill(gpu, nh, nkv, hd, block, base, n):
    rng = np.random.default_rng(base + 31 * n + nh)
    c = filled(rng, nkv, hd, block, base + n)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    want, bound = K.attention(q, c, base, 1 / math.sqrt(hd))
    close(attend(gpu, c, q, base, 1 / math.sqrt(hd)), want, bound)


def test_prefill_deep_and_rerun(gpu):
    rng = np.random.default_rng(11)
    c = filled(rng, 4, 256, 64, 5003)
    q = rng.standard_normal((43, 24, 256)).astype(np.float32)
    want, bound = K.attention(q, c, 4960, 1 / 16)
    got = attend(gpu, c, q, 4960, 1 / 16)
    close(got, want, bound)
    assert np.array_equal(got, attend(gpu, c, q, 4960, 1 / 16))


@pytest.mark.parametrize("entry", ["decode", "prefill"])
def test_q_stride(gpu, entry):
    rng = np.random.default_rng(5)
    c = filled(rng, 2, 64, 32, 70)
    for qs in (128, 65):
        q = rng.standard_normal((1 if entry == "decode" else 9, 6, 64)).astype(np.float32)
        base = 70 - len(q)
        want, bound = K.attention(q, c, base, 0.125)
        close(attend(gpu, c, q, base, 0.125, entry, qs), want, bound)


def test_no_key_gives_zeros(gpu):
    c = K.Cache(2, 64, 16, 16)
    with Bufs(gpu) as buf:
        out = buf(np.full(4 * 64, np.nan, np.float32))
        gpu.attn_decode_kv8(buf(np.ones(4 * 64, np.float32)), buf(c.codes), buf(c.scales), out, [4, 2, 64, 0, 64, F(1.0), 16])
        assert (out.array == 0).all()


@pytest.mark.parametrize("n", [1, 40])
def test_scales_far_apart(gpu, n):
    """Blocks whose scales differ by many powers of two, blocks of zeros, one key far above the rest."""
    rng = np.random.default_rng(n)
    seq = 300
    c = filled(rng, 2, 128, 16, seq)
    nb = c.scales.shape[0]
    c.scales[:, :, 1] = 2.0 ** rng.integers(-40, 9, (nb, 2))
    c.scales[3, :, 1] = 0
    c.scales[5] = 0
    c.codes[3, :, 1], c.codes[5] = 0, 0
    c.scales[7, :, 0] *= 30
    q = (rng.standard_normal((n, 4, 128)) * np.exp(rng.standard_normal((n, 4, 1)) * 2)).astype(np.float32)
    want, bound = K.attention(q, c, seq - n, 1 / math.sqrt(128))
    close(attend(gpu, c, q, seq - n, 1 / math.sqrt(128), "decode" if n == 1 else "prefill"), want, bound)


@pytest.mark.parametrize("n", [1, 40])
def test_values_all_tiny_or_all_zero(gpu, n):
    rng = np.random.default_rng(n)
    for vs in (2.0 ** -70, 0.0):
        c = filled(rng, 1, 64, 32, 100)
        c.scales[:4, :, 1] = vs
        q = rng.standard_normal((n, 3, 64)).astype(np.float32)
        want, bound = K.attention(q, c, 100 - n, 0.125)
        got = attend(gpu, c, q, 100 - n, 0.125, "decode" if n == 1 else "prefill")
        assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("n", [1, 40])
def test_nan_in_the_cache_reaches_only_who_reads_it(gpu, n):
    """A poisoned block makes every token that sees some of it NaN, in its head alone; q's NaN its row."""
    rng = np.random.default_rng(n)
    seq = 200
    for half in range(2):
        c = filled(rng, 2, 64, 16, seq)
        c.scales[11, 1, half] = np.nan                      # positions 176 .. 191
        q = rng.standard_normal((n, 4, 64)).astype(np.float32)
        q[n - 1, 0, 7] = np.inf if half else np.nan
        got = attend(gpu, c, q, seq - n, 0.125, "decode" if n == 1 else "prefill")
        c.scales[11, 1, half] = 0.01
        want, bound = K.attention(np.where(np.isfinite(q), q, 0), c, seq - n, 0.125)
        for t in range(n):
            sees = seq - n + t >= 176
            assert np.isnan(got[t, 2:]).all() == sees
            if not sees:
                close(got[t, 2:], want[t, 2:], bound[t, 2:])
            close(got[t, 1:2], want[t, 1:2], bound[t, 1:2])
        assert np.isnan(got[n - 1, 0]).all()


def test_two_handles_in_turn(gpu):
    """Two sg_gpu, each with a stream and scratch of its own, in turn and with sizes that regrow scratch."""
    rng = np.random.default_rng(8)
    with S.Gpu() as other:
        for seq in (40, 5000, 300, 9000):
            c = filled(rng, 2, 128, 32, seq)
            q = rng.standard_normal((1, 8, 128)).astype(np.float32)
            want, bound = K.attention(q, c, seq - 1, 0.09)
            a, b = (attend(g, c, q, seq - 1, 0.09, "decode") for g in (gpu, other))
            close(a, want, bound)
            assert np.array_equal(a, b)


def test_two_handles_at_once(gpu):
    """Two sg_gpu, a thread each, calls of several kinds side by side: every result is the one of the call alone."""
    import threading
    rng = np.random.default_rng(88)
    work = []
    for seq in (700, 5000, 33, 9000):
        c = filled(rng, 2, 128, 32, seq)
        q = rng.standard_normal((1, 8, 128)).astype(np.float32)
        work.append((c, q, seq, attend(gpu, c, q, seq - 1, 0.09, "decode")))
    wrong = []

    def run(g, order):
        for k in range(12):
            c, q, seq, want = work[order[k % 4]]
            if not np.array_equal(attend(g, c, q, seq - 1, 0.09, "decode"), want):
                wrong.append(seq)

    with S.Gpu() as other:
        threads = [threading.Thread(target=run, args=a) for a in ((gpu, (0, 1, 2, 3)), (other, (3, 2, 1, 0)))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not wrong


def test_cache_past_32_bits(gpu):
    """A cache of more than 4 GiB: rows behind the 32-bit line are stored, read back and attended to
    (the positions before hold zeros)."""
    nkv, hd, block, cap = 16, 256, 128, 560000
    L = S.lib()
    nb, ns = L.sg_kv8_code_bytes(nkv, hd, cap), L.sg_kv8_scale_bytes(nkv, block, cap)
    assert nb > 1 << 32

    class Wrapped:              # the device memory of an allocation, without its host mirror
        def __init__(self, nbytes):
            self.owner, self.handle = C.c_void_p(), C.c_void_p()
            S.check(L.sg_gpu_alloc(gpu.handle, nbytes, C.byref(self.owner), None))
            S.check(L.sg_gpu_wrap_device(gpu.handle, L.sg_gpu_buf_device(self.owner), nbytes, C.byref(self.handle)))

        def free(self):
            L.sg_gpu_buf_free(self.handle)
            L.sg_gpu_buf_free(self.owner)

    rng = np.random.default_rng(3)
    n, base = 9, cap - 9
    k, v = rows(rng, n, nkv, hd)
    q = rng.standard_normal((nkv * 2, hd)).astype(np.float32)
    codes, scales = Wrapped(nb), Wrapped(ns)
    with Bufs(gpu) as buf:
        bk, bv, out = buf(np.zeros_like(k)), buf(np.zeros_like(v)), buf(np.zeros_like(q))
        gpu.kv8_store(buf(k), buf(v), codes, scales, [nkv, hd, block, base, n])
        gpu.kv8_load(codes, scales, bk, bv, [nkv, hd, block, base, n])
        for got, x in ((bk.array, k), (bv.array, v)):
            step = np.abs(x).max(axis=(0, 2)) / 127
            assert (np.abs(got - x) <= 0.501 * step[None, :, None]).all()
        scale = 3.0 / 16            # scores far enough apart that the nine rows count beside the zeros
        gpu.attn_decode_kv8(buf(q), codes, scales, out, [nkv * 2, nkv, hd, cap, hd, F(scale), block])
        for h in range(nkv * 2):
            s = bk.array[:, h // 2].astype(np.float64) @ q[h].astype(np.float64) * scale
            m = max(s.max(), 0.0)
            p = np.exp(s - m)
            want = p @ bv.array[:, h // 2].astype(np.float64) / (p.sum() + (cap - n) * math.exp(-m))
            bound = (2 * (64 * np.abs(s).max() + 6) + cap / 16 + 64) * 2.0 ** -24 * np.abs(bv.array).max()
            assert (np.abs(out.array[h] - want) <= bound).all()
    codes.free()
    scales.free()


# ---------------------------------------------------------------- sizes past the small-call form

@pytest.mark.parametrize("nh,nkv,hd,block,base,n", [
    (24, 4, 256, 64, 3001, 203), (32, 8, 128, 16, 3000, 301), (12, 12, 64, 32, 8000, 401), (16, 1, 256, 128, 0, 800),
    (6, 2, 256, 64, 20000, 121), (10, 2, 128, 32, 15, 1500), (16, 1, 256, 128, 0, 1000), (8, 4, 64, 16, 6000, 1003),
    (5, 1, 64, 64, 30000, 310)])
def test_prefill_tiles(gpu, nh, nkv, hd, block, base, n):
    rng = np.random.default_rng(n)
    c = filled(rng, nkv, hd, block, base + n)
    q = rng.standard_normal((n, nh, hd)).astype(np.float32)
    want, bound = K.attention(q, c, base, 1 / math.sqrt(hd))
    got = attend(gpu, c, q, base, 1 / math.sqrt(hd))
    close(got, want, bound)
    assert np.array_equal(got, attend(gpu, c, q, base, 1 / math.sqrt(hd)))


def test_prefill_tiles_scales_and_nan(gpu):
    """The tile form on scales far apart, blocks of zeros, a poisoned block that only the last tokens see, and
    rows of q that are not finite, zero, or near the ends of the range."""
    rng = np.random.default_rng(21)
    seq, n, nh, hd = 6000, 128, 16, 256
    c = filled(rng, 1, hd, 16, seq)
    nb = -(-seq // 16)
    c.scales[:nb, :, 1] = 2.0 ** rng.integers(-40, 9, (nb, 1))
    c.scales[3, :, 1], c.scales[5] = 0, 0
    c.codes[3, :, 1], c.codes[5] = 0, 0
    c.scales[7, :, 0] *= 30
    c.scales[-(-seq // 16) - 4] = np.nan                        # positions 5936 .. 5951
    q = (rng.standard_normal((n, nh, hd)) * np.exp(rng.standard_normal((n, nh, 1)) * 2)).astype(np.float32)
    q[3, 2, 9], q[4, 5, 200], q[5, 1] = np.nan, -np.inf, 0
    q[6, 0] *= 1e-30
    q[7, 0] *= 1e-42
    got = attend(gpu, c, q, seq - n, 1 / 16)
    sees = seq - n + np.arange(n) >= 5936
    assert np.isnan(got[sees]).all() and sees.any() and not sees.all()
    bad = ~np.isfinite(q).all(axis=2)
    assert np.isnan(got[bad]).all()
    c.scales[-(-seq // 16) - 4] = 0.01
    want, bound = K.attention(np.where(np.isfinite(q), q, 0), c, seq - n, 1 / 16)
    ok = ~bad & ~sees[:, None]
    close(got[ok], want[ok], bound[ok])


@pytest.mark.parametrize("n,seq", [(1, 500), (30, 500), (128, 6000)])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_scale_of_either_sign(gpu, n, seq, scale):
    rng = np.random.default_rng(n)
    c = filled(rng, 1, 256, 32, seq)
    q = rng.standard_normal((n, 16, 256)).astype(np.float32)
    want, bound = K.attention(q, c, seq - n, float(np.float32(scale)))
    close(attend(gpu, c, q, seq - n, scale), want, bound)


@pytest.mark.parametrize("nh,nkv,hd,seq,n", [(24, 4, 256, 20011, 1), (8, 2, 128, 9001, 3), (12, 12, 64, 20011, 1), (8, 1, 256, 20001, 128)])
def test_values_that_cancel(gpu, nh, nkv, hd, seq, n):
    """Nearly flat weights over values without a mean: an output is the small remainder of a long sum, and has to
    be right by its own size. The weights' errors e (twice a score's, which the oracle's bound gives, and 10 u for exp
    and p s_V in two halves) and the additions' (m / 16 of them, each u of a partial sum that is no larger than the
    remainder) are independent of the values, so they add as squares: e + u sqrt(m / 16), doubled."""
    rng = np.random.default_rng(seq + n)
    c = filled(rng, nkv, hd, 64, seq)
    q = (rng.standard_normal((n, nh, hd)) * 0.01).astype(np.float32)
    scale = 1 / math.sqrt(hd)
    want, _ = K.attention(q, c, seq - n, scale)
    got = attend(gpu, c, q, seq - n, scale, "decode" if n == 1 else "prefill").astype(np.float64)
    u = 2.0 ** -24
    k = c.values(0, seq)
    most = max(np.abs(k[:, h] @ q[:, g].astype(np.float64).T).max() for g in range(nh) for h in [g * nkv // nh]) * scale
    ds = scale * 2 * u * np.abs(q).max() * np.abs(k).sum(2).max() + 16 * u * most
    tol = 2 * (2 * ds + 10 * u + u * math.sqrt(seq / 16))
    err = np.linalg.norm(got - want, axis=2) / np.linalg.norm(want, axis=2)
    assert (err <= tol).all(), f"worst error {err.max():.3g}, tolerance {tol:.3g}"
