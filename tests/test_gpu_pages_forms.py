"""The forms that the paged cache's operators take by size: eviction of a few rows, of many, of slots that do not
fit into LDS, of keys that crowd at the border; attention over one part and hundreds, over one sequence and more than
a wave has lanes."""
import numpy as np
import pytest

import pages_oracle as P
from test_gpu_pages import check_attn, check_evict, marks, pools, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("over", [1, 2, 3, 7, 8, 9, 10, 16, 17, 40])
@pytest.mark.parametrize("keep", [1, 5, 64, 1000])
@pytest.mark.parametrize("kind", ["ties", "apart", "zero", "nan"])
def test_evict_few_rows_too_many(gpu, over, keep, kind):
    """One by one up to eight, by the border past that; the lowest rows anywhere, among the newest slots too."""
    rng = np.random.default_rng(over * 31 + keep)
    table, pages = tables(rng, 3, -(-(keep + over) // 16) + 4)
    kp, vp = pools(rng, pages, 16, 2, 64)
    cap = table.shape[1] * 16
    weight, pos = marks(rng, 3, 2, cap, ties=kind == "ties")
    if kind == "zero":
        weight[...] = 0
    if kind == "nan":
        weight[rng.random(weight.shape) < 0.1] = np.nan
    for recent in (0, min(keep, 3), keep):
        check_evict(gpu, kp, vp, table, [keep + over, keep, keep + max(1, over // 2)], weight, pos, keep, recent)


@pytest.mark.parametrize("length,keep", [(3000, 1500), (5000, 4900), (32896, 1000), (32897, 32000), (40000, 20000), (66000, 100)])
@pytest.mark.parametrize("kind", ["crowd", "alike", "two", "spread", "signs"])
def test_evict_borders(gpu, length, keep, kind):
    """Keys that share their upper bits with the border (past what is listed of them), one key, two, all kinds; slots in LDS and
    more than fit there; marks in one round of the workgroup's and in several."""
    rng = np.random.default_rng(length + keep)
    table, pages = tables(rng, 1, -(-length // 256))
    kp, vp = pools(rng, pages, 256, 1, 64)
    weight, pos = marks(rng, 1, 1, table.shape[1] * 256, ties=False)
    u = rng.random(weight.shape).astype(np.float32)
    if kind == "crowd":
        weight = 1 + u / 8
    elif kind == "alike":
        weight[...] = 0.75
    elif kind == "two":
        weight = np.where(u < 0.4, 2.0, 2.0000002).astype(np.float32)
    elif kind == "signs":
        weight = (weight * np.where(u < 0.5, -1, 1)).astype(np.float32)
    for recent in (0, 77):
        check_evict(gpu, kp, vp, table, [length], weight, pos, keep, recent)


@pytest.mark.parametrize("keep", [63, 64, 65, 127, 128, 1023, 1024, 1025])
def test_evict_keep_at_the_edges(gpu, keep):
    rng = np.random.default_rng(keep)
    table, pages = tables(rng, 2, 20)
    kp, vp = pools(rng, pages, 64, 1, 64)
    weight, pos = marks(rng, 2, 1, 1280)
    check_evict(gpu, kp, vp, table, [1280, 1279], weight, pos, keep, keep // 3)


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 130])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (6, 1, 128), (2, 2, 256)])
def test_attn_by_number_of_sequences(gpu, n, nh, nkv, hd):
    """Up to 64 a wave finds its own part, past that a plan does; one long sequence among short and empty ones, at every place."""
    rng = np.random.default_rng(n + hd)
    for long in {0, n // 2, n - 1}:
        lens = rng.integers(0, 40, n)
        lens[long] = 1500
        table, pages = tables(rng, n, 47)
        kp, vp = pools(rng, pages, 32, nkv, hd)
        check_attn(gpu, rng.standard_normal((n, nh, hd)).astype(np.float32), kp, vp, table, lens, weights=True)


@pytest.mark.parametrize("n", [1, 3, 70])
def test_attn_of_nothing(gpu, n):
    rng = np.random.default_rng(n)
    table, pages = tables(rng, n, 3)
    kp, vp = pools(rng, pages, 16, 2, 64)
    got, _ = check_attn(gpu, rng.standard_normal((n, 4, 64)).astype(np.float32), kp, vp, table, [0] * n, rng.random((n, 2, 48)).astype(np.float32))
    assert not got.any()


@pytest.mark.parametrize("nh,nkv,hd,lens", [(16, 1, 64, [33000]), (16, 1, 128, [40000, 17]), (16, 1, 256, [30000]), (4, 4, 64, [12000, 9, 5000])])
def test_attn_of_many_parts(gpu, nh, nkv, hd, lens):
    """Hundreds of parts a sequence: more than a wave has lanes, than the join has in hand at once."""
    rng = np.random.default_rng(hd)
    n = len(lens)
    table, pages = tables(rng, n, -(-max(lens) // 256))
    kp, vp = pools(rng, pages, 256, nkv, hd)
    check_attn(gpu, rng.standard_normal((n, nh, hd)).astype(np.float32), kp, vp, table, lens, weights=True)


def test_attn_cancelling_values(gpu):
    """Weights nearly flat over values that cancel: what is left is what the sums' precision leaves."""
    rng = np.random.default_rng(1)
    table, pages = tables(rng, 1, 64)
    kp, vp = pools(rng, pages, 128, 1, 64, 1e-3)
    vp[...] = 1000.0
    vp[table[0, ::2]] = -1000.0
    check_attn(gpu, rng.standard_normal((1, 6, 64)).astype(np.float32), kp, vp, table, [8192], weights=True)


def test_attn_maximum_late_and_early(gpu):
    """The largest score in the first slot, the last, and rising all along: the running maximum's renewals."""
    rng = np.random.default_rng(2)
    table, pages = tables(rng, 3, 32)
    kp, vp = pools(rng, pages, 64, 1, 128, 0.1)
    q = np.ones((3, 4, 128), np.float32)
    for s, at in ((0, [0]), (1, [2047]), (2, range(0, 2048, 5))):
        for i, j in enumerate(at):
            kp[P.where(table, pages, 64, s, j)] = 1.0 + i / 64
    check_attn(gpu, q, kp, vp, table, [2048] * 3, weights=True)
