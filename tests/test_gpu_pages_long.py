"""Eviction of long rows: several workgroups a row (24576 slots and more, few rows), one a row (many rows) with the keys in LDS and
without, and calls of unlike forms that share a handle's scratch memory."""
import numpy as np
import pytest

from test_gpu_pages import check_evict, marks, pools, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [65, 4095, 4096, 4097, 12000, 28671, 30000, 40900])
@pytest.mark.parametrize("kind", ["spread", "crowd", "alike", "two", "halves", "odd"])
def test_evict_parts_of_a_row(gpu, keep, kind):
    """Lengths at the parts' edges (4096 slots), short and empty sequences beside them; keys that crowd at the border, alike ones
    over all parts, the lowest or the highest all in one part, weights of every kind."""
    rng = np.random.default_rng(keep)
    page = 64
    table, pages = tables(rng, 8, 640)
    kp, vp = pools(rng, 8, page, 1, 64)
    table = np.where(table < 8, table, -1).astype(np.int32)         # all but a few pages are not there: their marks move all the same
    cap = 640 * page
    weight, pos = marks(rng, 8, 1, cap, ties=False)
    u = rng.random(weight.shape).astype(np.float32)
    if kind == "crowd":
        weight = 1 + u / 8
    elif kind == "alike":
        weight[...] = 0.75
    elif kind == "two":
        weight = np.where(u < 0.4, 2.0, 2.0000002).astype(np.float32)
    elif kind == "halves":
        weight[:4, :, : cap // 2] += 1e6
        weight[4:, :, cap // 2 :] += 1e6
    elif kind == "odd":
        weight = np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, 3.4e38, -1.0], np.float32)[rng.integers(0, 8, weight.shape)]
        pos = rng.permutation(pos.ravel()).reshape(pos.shape)
    lens = [cap, cap - 1, 32768, 32769, 4096, 4097, 0, keep + 1]
    for recent in (0, min(keep, 100), keep):
        check_evict(gpu, kp, vp, table, lens, weight, pos, keep, recent)


@pytest.mark.parametrize("nkv,hd,page", [(3, 128, 32), (2, 256, 256)])
@pytest.mark.parametrize("length,keep", [(24576, 3000), (30011, 15000), (24575, 24000)])
def test_evict_parts_of_several_heads(gpu, nkv, hd, page, length, keep):
    rng = np.random.default_rng(length + hd)
    table, pages = tables(rng, 2, -(-length // page) + 1)
    kp, vp = pools(rng, pages, page, nkv, hd)
    weight, pos = marks(rng, 2, nkv, table.shape[1] * page)
    check_evict(gpu, kp, vp, table, [length, length - 300], weight, pos, keep, 99)


@pytest.mark.parametrize("length,keep", [(25000, 7000), (32896, 32000), (33000, 70), (42000, 30000), (42000, 41999)])
def test_evict_many_long_rows(gpu, length, keep):
    """Rows enough to fill the machine with a workgroup each; the keys in LDS up to 32896 slots, read again past that."""
    rng = np.random.default_rng(length)
    page, nkv = 256, 61
    table, pages = tables(rng, 1, -(-length // page))
    kp, vp = pools(rng, pages, page, nkv, 64) if length < 26000 else pools(rng, 2, page, nkv, 64)
    table = np.where(table < kp.shape[0], table, -1).astype(np.int32)
    weight, pos = marks(rng, 1, nkv, table.shape[1] * page)
    check_evict(gpu, kp, vp, table, [length], weight, pos, keep, min(keep, 64))


def test_evict_forms_in_turn(gpu):
    """A long row, short rows and a long row again: what one call left in the scratch memory does not reach the next."""
    rng = np.random.default_rng(9)
    table, pages = tables(rng, 1, 520)
    kp, vp = pools(rng, pages, 64, 1, 64)
    short, few = tables(rng, 3, 40)
    ks, vs = pools(rng, few, 64, 1, 64)
    for i in range(3):
        weight, pos = marks(rng, 1, 1, 520 * 64, ties=i == 1)
        check_evict(gpu, kp, vp, table, [33280 - 5000 * i], weight, pos, 4000 + i, 100)
        weight, pos = marks(rng, 3, 1, 40 * 64)
        check_evict(gpu, ks, vs, short, [2560, 100, 2000], weight, pos, 500, 100)
