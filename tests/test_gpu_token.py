"""Rotary positions with axes, token counts and processed logits on the GPU
against plain 64-bit forms, and one decoder's run of them with the 8-bit cache
between (include/surge.h)."""
import math

import numpy as np
import pytest

import kv8_oracle as K
import surge_amd as S
from test_gpu_kv8 import Bufs, close

pytestmark = pytest.mark.gpu
F = S.fbits
THETA = 1e7


def pack(sections, order):
    return sections[0] | sections[1] << 8 | sections[2] << 16 | order << 24


def rope(gpu, x, pos, rd, sections, order, stride=0, row=0, theta=THETA, in_place=False):
    n, nh, hd = x.shape
    hs, rw = stride or hd, row or nh * (stride or hd)
    full = np.full(((n - 1) * rw + (nh - 1) * hs + hd,), 9.0, np.float32)
    at = (np.arange(n)[:, None, None] * rw + np.arange(nh)[:, None] * hs + np.arange(hd)).astype(np.int64)
    full[at] = x
    with Bufs(gpu) as buf:
        b = buf(full)
        out = b if in_place else buf(np.full(full.shape, 5.0, np.float32))
        gpu.rope_axes(b, buf(pos.astype(np.int32)), out, [hd, rd, nh, stride, n, pack(sections, order), F(theta), row])
        got = out.array.copy()
    gaps = np.ones(full.shape, bool)
    gaps[at] = False
    assert (got[gaps] == (9.0 if in_place else 5.0)).all()      # gaps are left as they were
    return got[at]


@pytest.mark.parametrize("hd,rd,sections,order", [(256, 64, (12, 10, 10), 1), (256, 64, (12, 10, 10), 0), (128, 128, (24, 20, 20), 0),
                                                  (128, 128, (24, 20, 20), 1), (64, 2, (1, 0, 0), 1), (64, 16, (3, 2, 3), 0),
                                                  (64, 16, (0, 8, 0), 0), (64, 64, (32, 0, 0), 1), (100, 36, (6, 6, 6), 1),
                                                  (37, 22, (5, 3, 3), 1), (256, 256, (44, 42, 42), 1), (6, 6, (1, 1, 1), 1)])
@pytest.mark.parametrize("n,nh", [(1, 1), (1, 24), (3, 5), (4, 2), (33, 7)])
def test_rope_axes(gpu, hd, rd, sections, order, n, nh):
    rng = np.random.default_rng(hd + rd + n)
    x = rng.standard_normal((n, nh, hd)).astype(np.float32)
    pos = rng.integers(-50, 300000, (3, n))
    want, bound = K.rope_axes(x, pos, rd, sections, order, THETA)
    for kw in ({}, {"in_place": True}, {"stride": hd + 4, "row": nh * (hd + 4) + 8}, {"stride": 2 * hd, "in_place": True},
               {"stride": hd + 1, "row": nh * (hd + 1) + 3}):
        got = rope(gpu, x, pos, rd, sections, order, **kw)
        assert (np.abs(got - want) <= bound).all()
        assert np.array_equal(got[:, :, rd:], x[:, :, rd:])


def test_rope_axes_text_is_plain_rope(gpu):
    """The three axes alike: what k_rope_heads gives for that position."""
    rng = np.random.default_rng(4)
    x = rng.standard_normal((1, 6, 128)).astype(np.float32)
    p = 70001
    w = p * THETA ** (-2.0 * np.arange(32) / 64)
    cs = np.concatenate([np.cos(w), np.sin(w)]).astype(np.float32)
    with Bufs(gpu) as buf:
        out = buf(np.zeros_like(x))
        gpu.run_op("k_rope_heads", buf(x), buf(cs), out, [128, 64, 6, 128])
        plain = out.array.copy()
    got = rope(gpu, x, np.full((3, 1), p), 64, (12, 10, 10), 1)
    assert (np.abs(got - plain) <= 4 * 2.0 ** -24 * np.abs(x).max() * 2).all()


def test_rope_axes_many_tokens_and_infinities(gpu):
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1030, 3, 64)).astype(np.float32)
    x[5, 1, 3], x[6, 0, 60] = np.inf, np.nan
    pos = rng.integers(0, 2 ** 31 - 1, (3, 1030))           # the largest positions
    with np.errstate(invalid="ignore"):
        want, bound = K.rope_axes(x, pos, 32, (6, 5, 5), 1, THETA)
    got = rope(gpu, x, pos, 32, (6, 5, 5), 1)
    fin = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), fin)
    assert (np.abs(got - want)[fin] <= bound[fin]).all()


# ---------------------------------------------------------------- counts

@pytest.mark.parametrize("n,vocab,rows", [(0, 5, 1), (1, 1, 1), (7, 100, 3), (5000, 37, 2), (300000, 151936, 1), (33, 65, 70)])
def test_token_counts(gpu, n, vocab, rows):
    rng = np.random.default_rng(n)
    ids = rng.integers(-3, vocab + 3, (rows, n)).astype(np.int32)       # some outside: skipped
    if n > 100:
        ids[0, :n // 2] = vocab // 2                                    # one id over and over
    first = rng.integers(0, 9, (rows, vocab)).astype(np.uint32)
    want = np.stack([np.bincount(r[(r >= 0) & (r < vocab)], minlength=vocab) for r in ids])
    with Bufs(gpu) as buf:
        b, c = (buf(ids) if n else None), buf(first)
        gpu.token_counts(b, c, [n, vocab, rows, 0])
        assert np.array_equal(c.array, first + want)
        gpu.token_counts(b, c, [n, vocab, rows, 1])
        assert np.array_equal(c.array, want)


# ---------------------------------------------------------------- logits

def logits_oracle(x, counts, bias, allowed, rep, freq, pres):
    rep, freq, pres = (float(np.float32(v)) for v in (rep, freq, pres))
    y = x.astype(np.float64)
    with np.errstate(invalid="ignore"):
        b = np.abs(y)
        if counts is not None:
            c = counts.astype(np.float64)
            y = np.where(c > 0, np.where(y > 0, y / rep, y * rep), y)
            b = np.maximum(np.abs(y), b) + c * abs(freq) + (c > 0) * abs(pres)
            y = y - c * freq - (c > 0) * pres
        if bias is not None:
            y = y + bias
            b = b + np.abs(bias)
        if allowed is not None:
            y = np.where(allowed, y, -np.inf)
    return y, b * 4 * 2.0 ** -24            # four roundings, each of at most the sum of the sizes


def bits(allowed):
    r, v = allowed.shape
    w = np.zeros((r, -(-v // 32)), np.uint64)
    for j in range(v):
        w[:, j // 32] |= allowed[:, j].astype(np.uint64) << np.uint64(j % 32)
    return w.astype(np.uint32)


def run_logits(gpu, x, counts, bias, allowed, rep=1.0, freq=0.0, pres=0.0, in_place=False):
    rows, vocab = x.shape
    with Bufs(gpu) as buf:
        lx = buf(x)
        out = lx if in_place else buf(np.full_like(x, 3.0))
        tok = buf(np.zeros(rows, np.uint32))
        mask = None
        if allowed is not None:
            w = bits(allowed)
            if vocab % 32:
                w[:, -1] |= np.uint32(0xFFFFFFFF << (vocab % 32) & 0xFFFFFFFF)      # bits past the vocabulary mean nothing
            mask = buf(w)
        gpu.logits(lx, buf(counts) if counts is not None else None, buf(bias) if bias is not None else None, mask, out, tok,
                   [vocab, rows, F(rep), F(freq), F(pres)])
        return out.array.copy(), tok.array.copy()


def check_logits(gpu, x, counts, bias, allowed, rep, freq, pres):
    want, bound = logits_oracle(x, counts, bias, allowed, rep, freq, pres)
    got, tok = run_logits(gpu, x, counts, bias, allowed, rep, freq, pres)
    fin = np.isfinite(want)
    assert np.array_equal(got[~fin], want[~fin].astype(np.float32), equal_nan=True)
    assert (np.abs(got - want)[fin] <= bound[fin]).all()
    for r in range(len(x)):         # the token is the lowest index of the largest of what came out
        best = np.where(np.isnan(got[r]), -np.inf, got[r])
        assert tok[r] == (0xFFFFFFFF if best.max() == -np.inf else best.argmax())
    again, tok2 = run_logits(gpu, x, counts, bias, allowed, rep, freq, pres, in_place=True)
    assert np.array_equal(got, again, equal_nan=True) and np.array_equal(tok, tok2)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 5), (2, 31), (1, 32), (3, 33), (1, 257), (2, 1024), (5, 4099), (1, 151936), (3, 50001)])
@pytest.mark.parametrize("what", ["plain", "counts", "bias", "mask", "all"])
def test_logits(gpu, rows, vocab, what):
    rng = np.random.default_rng(vocab + rows)
    x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
    counts = rng.poisson(0.5, (rows, vocab)).astype(np.uint32) if what in ("counts", "all") else None
    bias = (rng.standard_normal(vocab) * 2).astype(np.float32) if what in ("bias", "all") else None
    allowed = rng.random((rows, vocab)) < 0.3 if what in ("mask", "all") else None
    check_logits(gpu, x, counts, bias, allowed, 1.3, 0.2, -0.4)


def test_logits_ties_infinities_and_nothing_allowed(gpu):
    vocab = 3001
    x = np.zeros((8, vocab), np.float32)
    x[0, [2999, 70, 700]] = 5.0                 # a tie: the lowest id
    x[1] = -np.inf                              # nothing above -inf
    x[2] = np.nan
    x[3, 17] = np.inf
    x[4, 5], x[4, 9] = np.nan, 1.0              # NaN is never chosen
    x[5] = -3e38
    x[6] = np.random.default_rng(0).standard_normal(vocab)
    x[7, :] = -np.inf
    x[7, 2222] = -3.4e38                        # the type's lowest value is above -inf
    allowed = np.ones((8, vocab), bool)
    allowed[6] = False                          # a mask that leaves nothing
    allowed[0, 70] = False
    check_logits(gpu, x, None, None, allowed, 1.0, 0.0, 0.0)
    _, tok = run_logits(gpu, x, None, None, allowed)
    none = 0xFFFFFFFF
    assert tok.tolist() == [700, none, none, 17, 9, 0, none, 2222]


@pytest.mark.parametrize("n", [0, 1, 3])
def test_what_lies_behind_an_output_stays(gpu, n):
    """Buffers larger than a call writes keep their ends, in the host's mirror too."""
    rng = np.random.default_rng(n)
    c = K.Cache(2, 64, 16, 64, rng)
    c.scales[...] = 0.01
    q = rng.standard_normal((max(n, 1), 4, 64)).astype(np.float32)
    with Bufs(gpu) as buf:
        out = buf(np.full((5, 4, 64), 7.0, np.float32))
        if n < 2:
            gpu.attn_decode_kv8(buf(q), buf(c.codes), buf(c.scales), out, [4, 2, 64, n * 40, 64, F(0.125), 16])
        else:
            gpu.attn_prefill_kv8(buf(q), buf(c.codes), buf(c.scales), out, [4, 2, 64, 40, n, 64, F(0.125), 16])
        assert (out.array[max(n, 1):] == 7.0).all() and (out.array[:max(n, 1)] != 7.0).all()
        x = rng.standard_normal((max(n, 1), 40)).astype(np.float32)
        o, token = buf(np.full((4, 40), 7.0, np.float32)), buf(np.full(6, 77, np.uint32))
        gpu.logits(buf(x), None, None, None, o, token, [40, max(n, 1), F(1.0), 0, 0, 0, 0, 0])
        assert (o.array[max(n, 1):] == 7.0).all() and np.array_equal(o.array[:max(n, 1)], x)
        assert (token.array[max(n, 1):] == 77).all() and np.array_equal(token.array[:max(n, 1)], x.argmax(1))
        k, v = (buf(np.full((4, 2, 64), 7.0, np.float32)) for _ in range(2))
        gpu.kv8_load(buf(c.codes), buf(c.scales), k, v, [2, 64, 16, 3, max(n, 1), 0, 0, 0])
        assert (k.array[max(n, 1):] == 7.0).all() and (v.array[max(n, 1):] == 7.0).all()
        counts = buf(np.full((4, 40), 3, np.uint32))
        gpu.token_counts(buf(np.zeros((max(n, 1), 5), np.int32)), counts, [5, 40, max(n, 1), 1])
        assert (counts.array[max(n, 1):] == 3).all() and (counts.array[:max(n, 1), 0] == 5).all() and not counts.array[:max(n, 1), 1:].any()


def test_logits_plain_is_the_argmax(gpu):
    rng = np.random.default_rng(9)
    x = rng.standard_normal((1, 151936)).astype(np.float32)
    with Bufs(gpu) as buf:
        t = buf(np.zeros(1, np.uint32))
        gpu.run_op("k_argmax", buf(x), None, t, [x.size])
        got, tok = run_logits(gpu, x, None, None, None)
        assert tok[0] == t.array[0] and np.array_equal(got, x)


# ---------------------------------------------------------------- a run of them together

@pytest.mark.parametrize("nh,nkv,hd,rd,sections,block,chunks", [(6, 2, 64, 32, (6, 5, 5), 32, (37, 20, 1, 1, 1)),
                                                                (12, 2, 256, 64, (12, 10, 10), 64, (70, 1, 1, 3))])
def test_a_sequence_through_all_of_them(gpu, nh, nkv, hd, rd, sections, block, chunks):
    """A prompt in chunks, then token by token: rotate q and k, store k and v in 8 bits, attend,
    choose a token under the counts of what was chosen; the cache's bits and every output against
    the plain forms on the same inputs."""
    rng = np.random.default_rng(hd)
    total, vocab = sum(chunks), 700
    pos = np.sort(rng.integers(0, 5000, (3, total)), axis=1)
    c = K.Cache(nkv, hd, block, total, rng)
    counts = np.zeros(vocab, np.uint32)
    head = (rng.standard_normal((nh * hd, vocab)) / math.sqrt(nh * hd)).astype(np.float32) * 8
    with Bufs(gpu) as buf:
        codes, scales, cnt = buf(c.codes), buf(c.scales), buf(counts)
        base = 0
        for n in chunks:
            q = rng.standard_normal((n, nh, hd)).astype(np.float32)
            k, v = rng.standard_normal((2, n, nkv, hd)).astype(np.float32)
            p = pos[:, base:base + n]
            sec = pack(sections, 1)
            bq, bk, bp = buf(q), buf(k), buf(p.astype(np.int32))
            gpu.rope_axes(bq, bp, bq, [hd, rd, nh, 0, n, sec, F(THETA)])
            gpu.rope_axes(bk, bp, bk, [hd, rd, nkv, 0, n, sec, F(THETA)])
            for got, x in ((bq.array, q), (bk.array, k)):
                want, bound = K.rope_axes(x, p, rd, sections, 1, THETA)
                assert (np.abs(got - want) <= bound).all()
            gpu.kv8_store(bk, buf(v), codes, scales, [nkv, hd, block, base, n])
            c.store(bk.array.copy(), v, base)
            assert np.array_equal(codes.array, c.codes) and np.array_equal(scales.array, c.scales)
            out = buf(np.zeros((n, nh, hd), np.float32))
            if n == 1:
                gpu.attn_decode_kv8(bq, codes, scales, out, [nh, nkv, hd, base + 1, hd, F(hd ** -0.5), block])
            else:
                gpu.attn_prefill_kv8(bq, codes, scales, out, [nh, nkv, hd, base, n, hd, F(hd ** -0.5), block])
            want, bound = K.attention(bq.array.copy(), c, base, hd ** -0.5)
            close(out.array, want, bound)
            x = (out.array[-1:].reshape(1, -1) @ head).astype(np.float32)
            lo, tok = buf(x), buf(np.zeros(1, np.uint32))
            gpu.logits(lo, cnt, None, None, lo, tok, [vocab, 1, F(1.5), F(0.3), F(0.1)])
            y, _ = logits_oracle(x, counts[None], None, None, 1.5, 0.3, 0.1)
            assert tok.array[0] == lo.array[0].argmax() and abs(y[0].max() - lo.array[0].max()) < 1e-4
            gpu.token_counts(tok, cnt, [1, vocab, 1, 0])
            counts[tok.array[0]] += 1
            assert np.array_equal(cnt.array, counts)
            base += n
