"""Token counts over several ranges of the vocabulary and in tables, and logits
whose threads take several steps: the forms that real vocabularies take."""
import numpy as np
import pytest

import surge_amd as S
from test_gpu_kv8 import Bufs
from test_gpu_token import logits_oracle

pytestmark = pytest.mark.gpu
F = S.fbits


# ---------------------------------------------------------------- counts

@pytest.mark.parametrize("n,vocab,rows", [(900, 151936, 1), (900, 151936, 16), (32000, 151936, 16), (131072, 8193, 1), (131072, 2048, 2),
                                          (131073, 2049, 3), (131073, 8193, 2), (5000, 20001, 40), (1, 524289, 1), (3000, 8192, 300)])
def test_token_counts_over_ranges(gpu, n, vocab, rows):
    """Ranges of 2048 ids, of 8192, and the tables past 131072 ids a row: ids at every range's edges, outside the
    vocabulary, alike neighbours, one id over and over; added and counted anew."""
    rng = np.random.default_rng(n + vocab)
    ids = rng.integers(-2, vocab + 2, (rows, n)).astype(np.int32)
    edges = np.unique([e + d for e in range(0, vocab + 8192, 2048) for d in (-1, 0, 1)])
    if n > 3 * len(edges):
        ids[:, 7:7 + 2 * len(edges):2] = edges
        ids[:, n // 2:] = np.repeat(ids[:, n // 2:], 3, axis=1)[:, :n - n // 2]        # threes
        ids[0, n // 3:n // 2] = vocab - 1
    elif n < 10:
        ids[...] = vocab - 1
    first = rng.integers(0, 9, (rows, vocab)).astype(np.uint32)
    want = np.stack([np.bincount(r[(r >= 0) & (r < vocab)], minlength=vocab) for r in ids])
    with Bufs(gpu) as buf:
        b, c = buf(ids), buf(first)
        gpu.token_counts(b, c, [n, vocab, rows, 0])
        assert np.array_equal(c.array, first + want)
        gpu.token_counts(b, c, [n, vocab, rows, 1])
        assert np.array_equal(c.array, want)


# ---------------------------------------------------------------- logits

@pytest.mark.parametrize("rows,vocab", [(24, 151936), (40, 151935), (1700, 4100), (3300, 2003)])
def test_logits_in_several_steps(gpu, rows, vocab):
    """More rows than the launch has workgroups for at a step each: 16-byte and single accesses, a few parts a row and
    one. The best ids lie in first, middle and last steps; ties go to the lowest."""
    rng = np.random.default_rng(rows)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    counts = rng.integers(0, 3, (rows, vocab)).astype(np.uint32)
    bias = rng.standard_normal(vocab).astype(np.float32)
    words = rng.integers(0, 1 << 32, (rows, -(-vocab // 32)), dtype=np.uint32)
    best = np.array([(vocab - 1 - 7 * r) % vocab if r % 3 == 0 else r * vocab // rows if r % 3 == 1 else r % vocab for r in range(rows)])
    r = np.arange(rows)
    for at in (best, np.minimum(best + vocab // 2, vocab - 1)):         # the second is a tie, or lower in the order
        x[r, at], counts[r, at] = 50.0, 0
        words[r, at // 32] |= np.uint32(1) << (at % 32).astype(np.uint32)
    bias[np.concatenate([best, np.minimum(best + vocab // 2, vocab - 1)])] = 0.5
    words[rows // 2] = 0                                                # a row with nothing allowed
    allowed = np.unpackbits(words.view(np.uint8), axis=1, bitorder="little")[:, :vocab].astype(bool)
    want, bound = logits_oracle(x, counts, bias, allowed, 1.3, 0.2, -0.4)
    with Bufs(gpu) as buf:
        out, tok = buf(np.full_like(x, 3.0)), buf(np.zeros(rows, np.uint32))
        gpu.logits(buf(x), buf(counts), buf(bias), buf(words), out, tok, [vocab, rows, F(1.3), F(0.2), F(-0.4)])
        got, token = out.array.copy(), tok.array.copy()
    assert np.array_equal(got[~allowed], want[~allowed].astype(np.float32))
    assert (np.abs(got[allowed] - want[allowed]) <= bound[allowed]).all()
    best[rows // 2] = -1
    assert np.array_equal(token.astype(np.int32), best)
