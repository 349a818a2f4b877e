"""Refusals of the paged cache's operators and of sampling. Every check precedes
the first use of the device, so they are tested here, on handles that wrap
addresses nothing will touch; and the plain forms' own rules."""
import numpy as np
import pytest

import pages_oracle as P
import surge_amd as S
from test_operators_host import AT, buf, far, refused

F = S.fbits
STORE, ATTN, EVICT, SAMPLE = ("sg_gpu_run_page_store", "sg_gpu_run_attn_paged", "sg_gpu_run_page_evict", "sg_gpu_run_sample")

# 2 kv heads x 64, pages of 16, 3 sequences of 4 pages, a pool of 14 pages
POOL, TABLE, SLOTS, ROWS = 14 * 16 * 2 * 64 * 2, 3 * 4 * 4, 3 * 2 * 64 * 4, 3 * 5 * 128 * 4


def store_bufs():
    return [far(ROWS), far(ROWS), far(POOL), far(POOL), far(TABLE), far(36), far(SLOTS), far(SLOTS)]


def attn_bufs():
    return [far(3 * 4 * 64 * 4), far(POOL), far(POOL), far(TABLE), far(12), far(SLOTS), far(SLOTS), far(3 * 4 * 64 * 4)]


def evict_bufs():
    return [far(POOL), far(POOL), far(TABLE), far(12)] + [far(SLOTS) for _ in range(4)]


def sample_bufs():
    return [far(3 * 100 * 4), far(48), far(12), far(12), far(3 * 100 * 4)]


PARAMS = {STORE: [2, 64, 16, 3, 4, 5, 0], ATTN: [4, 2, 64, 16, 3, 4, 64, F(0.125)], EVICT: [2, 64, 16, 3, 4, 40, 8], SAMPLE: [100, 3]}
BUFS = {STORE: store_bufs, ATTN: attn_bufs, EVICT: evict_bufs, SAMPLE: sample_bufs}


def changed(name, change):
    p = list(PARAMS[name])
    for i, v in change.items():
        p[i] = v
    return p


@pytest.mark.parametrize("name,change,match", [
    (STORE, {0: 0}, "n_kv"), (STORE, {0: 65536}, "n_kv"), (STORE, {1: 96}, "head_dim"), (STORE, {2: 8}, "page 16"), (STORE, {2: 48}, "page 16"),
    (STORE, {2: 512}, "page 16"), (STORE, {3: 0}, "n_seq"), (STORE, {3: 32769}, "n_seq"), (STORE, {4: 0}, "slots"), (STORE, {4: 1 << 27}, "slots"),
    (STORE, {4: 0xFFFFFFFF}, "slots"), (STORE, {3: 4}, "table holds"), (STORE, {4: 5}, "table holds"), (STORE, {2: 256, 1: 128}, "kp holds"),
    (STORE, {5: 0}, "n must"), (STORE, {5: (1 << 27) + 1}, "n must"), (STORE, {5: 6}, "k holds"), (STORE, {6: 127}, "stride"),
    (STORE, {6: 129}, "k holds"), (STORE, {3: 32768, 4: 1, 5: 1 << 27, 6: 0xFFFFFFFF}, "table holds"),
    (ATTN, {0: 0}, "n_heads"), (ATTN, {0: 5}, "n_heads"), (ATTN, {0: 34}, "n_heads"), (ATTN, {1: 0}, "n_kv"), (ATTN, {2: 32}, "head_dim"),
    (ATTN, {3: 17}, "page 16"), (ATTN, {4: 0}, "n_seq"), (ATTN, {5: 0}, "slots"), (ATTN, {5: 5}, "table holds"), (ATTN, {6: 63}, "q_stride"),
    (ATTN, {6: 65}, "q holds"), (ATTN, {6: 0xFFFFFFFF}, "q holds"), (ATTN, {0: 8}, "q holds"),
    (EVICT, {0: 0}, "n_kv"), (EVICT, {1: 0}, "head_dim"), (EVICT, {2: 0}, "page 16"), (EVICT, {3: 0}, "n_seq"), (EVICT, {4: 5}, "table holds"),
    (EVICT, {5: 0, 6: 0}, "keep"), (EVICT, {6: 41}, "recent"),
    (SAMPLE, {0: 0}, "vocab"), (SAMPLE, {0: 1 << 31}, "vocab"), (SAMPLE, {1: 0}, "rows"), (SAMPLE, {1: 65536}, "rows"),
    (SAMPLE, {0: 101}, "logits holds"), (SAMPLE, {1: 4}, "logits holds")])
def test_bad_shapes_are_refused(name, change, match):
    refused(name, BUFS[name](), changed(name, change), match)


@pytest.mark.parametrize("name", [STORE, ATTN, EVICT, SAMPLE])
def test_null_short_and_misaligned_buffers_are_refused(name):
    may_be_none = {STORE: (6, 7), ATTN: (5,), EVICT: (), SAMPLE: (4,)}[name]
    sizes = {STORE: [ROWS, ROWS, None, None, TABLE, 36, SLOTS, SLOTS], ATTN: [3 * 4 * 64 * 4, None, None, TABLE, 12, SLOTS, SLOTS, 3 * 4 * 64 * 4],
             EVICT: [None, None, TABLE, 12, SLOTS, SLOTS, SLOTS, SLOTS], SAMPLE: [1200, 48, 12, 12, 1200]}[name]
    p = PARAMS[name]
    refused(name, BUFS[name](), None, "NULL")
    for i, size in enumerate(sizes):
        h = BUFS[name]()
        if i not in may_be_none:
            keep = h[i]
            h[i] = None
            refused(name, h, p, "weight_out" if (name, i) == (ATTN, 6) else "NULL")
            h[i] = keep
        if size is None:            # a pool: not one whole page
            h[i] = far(16 * 2 * 64 * 2 - 1)
            refused(name, h, p, "holds")
            h[i] = buf(POOL, (AT << 1) + 8)
        else:
            h[i] = far(size - 1)
            refused(name, h, p, "holds")
            h[i] = buf(size, (AT << 1) + 2)
        refused(name, h, p, "aligned")


def test_overlapping_buffers_are_refused():
    def both(name, i, j, off=0, p=None):
        """Buffer j moved onto i's memory, `off` bytes behind its start."""
        h = BUFS[name]()
        h[i], h[j] = buf(1 << 20, AT << 2), buf(1 << 20, (AT << 2) + off)
        refused(name, h, p or PARAMS[name], "overlap")

    for j in (3, 4, 5, 6, 7):
        both(STORE, 2, j)
    for i, j in ((0, 2), (1, 2), (0, 3), (1, 3), (0, 6), (0, 7), (4, 6), (5, 7), (6, 7), (3, 4), (3, 5)):
        both(STORE, i, j)
    for i, j in ((0, 7), (1, 7), (2, 7), (3, 7), (4, 7), (6, 7), (5, 7), (0, 6), (1, 6), (2, 6), (3, 6), (4, 6), (1, 2), (1, 3), (2, 3)):
        both(ATTN, i, j)
    both(ATTN, 5, 6, 16)
    for i, j in ((0, 1), (0, 2), (1, 2), (0, 3), (1, 3), (0, 4), (1, 5), (0, 6), (2, 6), (3, 6), (2, 7), (3, 7), (4, 7), (5, 6), (6, 7)):
        both(EVICT, i, j)
    both(EVICT, 4, 6, 16)
    both(EVICT, 5, 7, 16)
    for i, j in ((0, 3), (1, 3), (2, 3), (3, 4), (1, 4), (2, 4)):
        both(SAMPLE, i, j)
    both(SAMPLE, 0, 4, 16)


def test_sizes_past_64_bits_are_refused():
    """32768 sequences of 65535 x 16 heads at the largest stride: 2^67 bytes, which would wrap to a size that fits."""
    h = [far(1 << 39), far(1 << 28), far(1 << 28), far(1 << 18), far(1 << 18), None, None, far(1 << 39)]
    refused(ATTN, h, [65535 * 16, 65535, 64, 16, 32768, 1, 0xFFFFFFFF, F(0.125)], "too large")


def test_plain_sampling_follows_its_rules():
    """A worked example: weights 4, 2, 2, 1, 1 of ten."""
    x = np.log(np.array([2.0, 1.0, 4.0, 2.0, 1.0]))
    t = lambda k, p, m, u: P.sample(x, 1.0, k, p, m, u)
    assert np.allclose(t(0, 1.0, 0.0, 0.0)[1] * 10, [2, 1, 4, 2, 1])
    assert [t(0, 1.0, 0.0, u)[0] for u in (0.0, 0.19, 0.21, 0.29, 0.31, 0.69, 0.71, 0.89, 0.91)] == [0, 0, 1, 1, 2, 2, 3, 3, 4]
    assert np.allclose(t(2, 1.0, 0.0, 0)[1] * 6, [2, 0, 4, 0, 0])             # of two alike the lower id
    assert np.allclose(t(0, 0.5, 0.0, 0)[1] * 6, [2, 0, 4, 0, 0])
    assert np.allclose(t(3, 0.49, 0.0, 0)[1], [0, 0, 1, 0, 0])                # half of eight is reached by the first
    assert np.allclose(t(0, 1.0, 0.4, 0)[1] * 8, [2, 0, 4, 2, 0])
    assert np.allclose(t(0, 0.0, 0.0, 0)[1], [0, 0, 1, 0, 0])
    assert P.sample(x, 0.0, 0, 1.0, 0.0, 0.9)[0] == 2


def test_plain_eviction_follows_its_rules():
    kp = np.arange(6, dtype=np.float16).reshape(6, 1, 1, 1) * np.ones((1, 1, 1, 2), np.float16)
    vp = -kp
    table = np.array([[5, 4, 3, 2, 1, 0]], np.int32)
    weight = np.array([[[3, 0, 1, 1, 2, 0]]], np.float32)
    pos = np.array([[[0, 1, 2, 5, 6, 9]]], np.int32)
    wo, po = P.evict(kp, vp, table, [6], weight, pos, 3, 1)
    assert po[0, 0, :3].tolist() == [0, 6, 9] and wo[0, 0, :3].tolist() == [3, 2, 0]      # the last, then weights 3 and 2
    assert kp[[5, 4, 3], 0, 0, 0].tolist() == [5, 1, 0]
