"""Every form of the attention over the 8-bit cache, at sizes that reach it (as
sg_gpu_attn_kv8_parts says), and a cache past 4 GiB in both of them."""
import ctypes as C
import math

import numpy as np
import pytest

import kv8_oracle as K
import surge_amd as S
from test_gpu_kv8 import Bufs, attend
from test_gpu_kv8_precision import plain

pytestmark = pytest.mark.gpu
F = S.fbits


def close_by_size(got, want, ds, keys, what):
    """Each output by its own norm: weights' errors e (a score's twice, 10 u) and the additions' (m / 16, each u of a
    partial sum no larger than the remainder) add as squares, doubled."""
    u = 2.0 ** -24
    tol = 2 * (2 * ds + 10 * u + u * np.sqrt(keys / 16)[:, None])
    err = np.linalg.norm(got - want, axis=2) / np.linalg.norm(want, axis=2) / tol
    assert (err <= 1).all(), f"{what}: worst error {err.max():.2f} of its tolerance"


@pytest.mark.parametrize("nh,nkv,hd,base,n,parts,waves", [
    (12, 12, 64, 100, 1, 1, 4), (24, 4, 256, 383, 1, 1, 8), (12, 12, 64, 300, 1, 1, 8), (16, 1, 128, 600, 1, 1, 8), (16, 1, 256, 0, 800, 1, 4),
    (8, 2, 256, 699, 1, 6, 4), (12, 12, 64, 2000, 1, 16, 4), (24, 4, 256, 17003, 1, 64, 4), (3, 1, 64, 33332, 1, 261, 4),
    (32, 8, 128, 8000, 40, 3, 8), (12, 12, 64, 12001, 60, 10, 8),
    (12, 12, 64, 0, 2500, 1, 0), (32, 8, 256, 0, 1024, 1, 0), (48, 8, 128, 0, 1024, 1, 0), (16, 1, 256, 0, 1000, 1, 0),
    (12, 12, 64, 8000, 500, 5, 0), (32, 8, 128, 3000, 301, 3, 0), (24, 4, 256, 3001, 203, 6, 0),
    (5, 1, 64, 30000, 310, 19, 0), (8, 1, 128, 20000, 130, 3, 8), (8, 1, 128, 20000, 200, 19, 0), (6, 2, 256, 20000, 121, 40, 0)])
def test_attention_forms(gpu, nh, nkv, hd, base, n, parts, waves):
    """One workgroup, parts joined by either join, and four or eight waves of each; tiles whole, joined by either."""
    assert gpu.attn_kv8_parts(nh, nkv, hd, base, n) == (parts, waves)
    rng = np.random.default_rng(base + n)
    m = base + n
    c = K.Cache(nkv, hd, 32, m)
    c.codes[...] = rng.integers(-127, 128, c.codes.shape)
    c.scales[...] = rng.uniform(0.005, 0.03, c.scales.shape)
    q = (rng.standard_normal((n, nh, hd)) * 0.3).astype(np.float32)
    want, ds = plain(q, c, base, 1 / math.sqrt(hd))
    got = attend(gpu, c, q, base, 1 / math.sqrt(hd), "decode" if n == 1 else "prefill")
    close_by_size(got, want, ds, np.arange(base + 1, m + 1), (parts, waves))
    assert np.array_equal(got, attend(gpu, c, q, base, 1 / math.sqrt(hd), "decode" if n == 1 else "prefill"))


@pytest.mark.parametrize("nh,nkv,hd,base,n", [(12, 12, 64, 8000, 500), (12, 12, 64, 0, 2500), (16, 2, 128, 9000, 600)])
def test_values_that_cancel_in_tiles(gpu, nh, nkv, hd, base, n):
    """Nearly flat weights over values without a mean, at the head dims whose tiles no other such test takes."""
    assert gpu.attn_kv8_parts(nh, nkv, hd, base, n)[1] == 0
    rng = np.random.default_rng(hd)
    m = base + n
    c = K.Cache(nkv, hd, 64, m)
    c.codes[...] = rng.integers(-127, 128, c.codes.shape)
    c.scales[...] = rng.uniform(0.005, 0.03, c.scales.shape)
    q = (rng.standard_normal((n, nh, hd)) * 0.01).astype(np.float32)
    want, ds = plain(q, c, base, 1 / math.sqrt(hd))
    close_by_size(attend(gpu, c, q, base, 1 / math.sqrt(hd)), want, ds, np.arange(base + 1, m + 1), "cancel")


class Raw:
    """Device memory of its own, without a host mirror, and views of it."""

    def __init__(self, gpu, nbytes):
        self.gpu, self.nbytes, self.owner, self.views = gpu, nbytes, C.c_void_p(), []
        S.check(S.lib().sg_gpu_alloc(gpu.handle, nbytes, C.byref(self.owner), None))
        self.handle = self.at(0).handle

    def at(self, off):
        v = type("View", (), {})()
        v.handle = C.c_void_p()
        S.check(S.lib().sg_gpu_wrap_device(self.gpu.handle, S.lib().sg_gpu_buf_device(self.owner) + off, self.nbytes - off, C.byref(v.handle)))
        self.views.append(v)
        return v

    def free(self):
        for v in self.views:
            S.lib().sg_gpu_buf_free(v.handle)
        S.lib().sg_gpu_buf_free(self.owner)


def test_cache_past_4_gib(gpu):
    """Rows whose codes lie past 2^32 bytes: stored, found at the address that the layout gives (a cache that starts
    there), and attended to by both forms, with queries along the stored keys, so that their few weights outweigh the
    half million zero keys before them."""
    nkv, hd, block, cap, rows = 16, 256, 128, 560000, 40
    L = S.lib()
    nb, ns = L.sg_kv8_code_bytes(nkv, hd, cap), L.sg_kv8_scale_bytes(nkv, block, cap)
    base = cap - rows
    first = base // block * block                       # a cache of its own from this position on
    assert first * nkv * 2 * hd > 1 << 32
    rng = np.random.default_rng(3)
    k, v = rng.standard_normal((2, rows, nkv, hd)).astype(np.float32)
    codes, scales = Raw(gpu, nb), Raw(gpu, ns)
    try:
        with Bufs(gpu) as buf:
            bk, bv = buf(np.zeros_like(k)), buf(np.zeros_like(v))
            gpu.kv8_store(buf(k), buf(v), codes, scales, [nkv, hd, block, base, rows])
            c = K.Cache(nkv, hd, block, cap - first)
            if base > first:
                c.store(np.zeros((base - first, nkv, hd), np.float32), np.zeros((base - first, nkv, hd), np.float32), 0)
            c.store(k, v, base - first)
            for co, sc, at in ((codes, scales, base), (codes.at(first * nkv * 2 * hd), scales.at(first // block * nkv * 8), base - first)):
                gpu.kv8_load(co, sc, bk, bv, [nkv, hd, block, at, rows])
                for got, half in ((bk.array, 0), (bv.array, 1)):
                    assert np.array_equal(got, c.values(half, cap - first)[base - first:].astype(np.float32))
            kd, vd = (c.values(half, cap - first)[base - first:] for half in range(2))
            for n, tiles in ((1, False), (17, True)):
                parts, waves = gpu.attn_kv8_parts(2 * nkv, nkv, hd, cap - n, n)
                assert (waves == 0) == tiles
                # a token's heads look for one row that it sees: scores of 25 there, of order 1.6 elsewhere
                pick = rng.integers(0, rows - n + 1, (n, 2 * nkv))
                q = np.stack([[kd[pick[t, h], h // 2] * (25 * 16 / (kd[pick[t, h], h // 2] ** 2).sum()) for h in range(2 * nkv)]
                              for t in range(n)]).astype(np.float32)
                out = buf(np.zeros((n, 2 * nkv, hd), np.float32))
                if n == 1:
                    gpu.attn_decode_kv8(buf(q), codes, scales, out, [2 * nkv, nkv, hd, cap, hd, F(1 / 16), block])
                else:
                    gpu.attn_prefill_kv8(buf(q), codes, scales, out, [2 * nkv, nkv, hd, cap - n, n, hd, F(1 / 16), block])
                for t in range(n):
                    sees = rows - n + 1 + t
                    for h in range(2 * nkv):
                        s = kd[:sees, h // 2] @ q[t, h].astype(np.float64) / 16
                        p = np.exp(s - s.max())
                        want = p @ vd[:sees, h // 2] / (p.sum() + (base) * np.exp(-s.max()))
                        assert np.linalg.norm(want) > 0.9 * np.linalg.norm(vd[pick[t, h], h // 2])
                        # the score's rounding twice, as the oracle's bound has it, and 10 u as there (the zero keys are 8e-6 of
                        # the sum, its 35000 additions of theirs u each at most: 0.3 u of the whole)
                        ds = 2 * 2.0 ** -24 * np.abs(q[t, h]).max() * np.abs(kd[:, h // 2]).sum(1).max() / 16 + 16 * 2.0 ** -24 * 25
                        err = np.linalg.norm(out.array[t, h] - want) / np.linalg.norm(want)
                        assert err <= 2 * (2 * ds + 10 * 2.0 ** -24)
    finally:
        codes.free()
        scales.free()
