"""Sampling where its rules meet: a floor for the weights that no id reaches, over ids that are alike (include/surge.h)."""
import numpy as np
import pytest

from test_gpu_sample import check, rows_of, sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("min_p", [np.float32(1) + np.float32(2.0 ** -23), 1.5, 1e30, np.inf])
@pytest.mark.parametrize("vocab", [4, 300, 5000, 151936])
def test_no_id_reaches_min_p(gpu, min_p, vocab):
    """A min_p above 1 leaves the largest alone, of alike ones the lowest id, whatever else is asked for."""
    rng = np.random.default_rng(vocab)
    x = np.minimum(rows_of(rng, 1, vocab, True), np.float32(2.0))       # many at 2
    x[0, :4] = [1, 3, 3, 0]
    x[0, vocab // 2] = x[0, vocab - 1] = 3.0
    y = x.copy()
    y[0, [2, vocab - 1]] = np.inf
    z = np.full_like(x, -1.25)
    sets = [(t, k, p, min_p) for t, k, p in ((1.0, 0, 1.0), (0.5, 3, 1.0), (1.0, 200, 1.0), (1.0, 0, 0.9), (2.0, 1000, 0.55), (0.0, 0, 1.0), (np.inf, 0, 1.0))]
    u = [0.0, 0.3, 0.9, 0.999, 0.5, 0.7, 0.6]
    for row, first in ((x, 1), (y, 2), (z, 0)):
        rows = np.repeat(row, len(sets), 0)
        tok, pr = check(gpu, rows, sets, u)
        assert (tok == first).all() and (pr.sum(axis=1) == 1.0).all()
        tok, _ = sample(gpu, rows, sets, u, probs=False)
        assert (tok == first).all()


def test_min_p_of_one_keeps_all_that_are_alike(gpu):
    x = np.array([[1, 3, 3, 0]], np.float32)
    tok, pr = sample(gpu, np.repeat(x, 3, 0), [(1.0, 0, 1.0, 1.0)] * 3, [0.2, 0.49, 0.6])
    assert tok.tolist() == [1, 1, 2] and pr[0].tolist() == [0, 0.5, 0.5, 0]
