"""Refusals of the 8-bit cache's, the several-axis rotary and the logits
operators, and their sizes. Every check precedes the first use of the device,
so they are tested here, on handles that wrap addresses nothing will touch."""
import ctypes as C
import math

import numpy as np
import pytest

import kv8_oracle as K
import surge_amd as S

G = C.create_string_buffer(8192)        # stands for a handle: a refused call does not look into it
AT = 0x7000_0000_0000
F = S.fbits


def buf(nbytes, at=AT):
    h = C.c_void_p()
    S.check(S.lib().sg_gpu_wrap_device(G, at, nbytes, C.byref(h)))
    return h


_next = [AT]


def far(nbytes):
    """A handle at an address of its own."""
    _next[0] += 1 << 40
    return buf(nbytes, _next[0])


def refused(name, handles, p, match):
    with pytest.raises(S.SurgeError, match=match):
        S.check(getattr(S.lib(), name)(G, *handles, S.params(p) if p is not None else None))


def test_layout_is_a_permutation_of_the_record():
    for hd in (64, 128, 256):
        for at in (K.key_at, K.val_at):
            idx = sorted(at(r, d) for r in range(16) for d in range(hd))
            assert idx == list(range(16 * hd))


def test_cache_sizes():
    L = S.lib()
    assert L.sg_kv8_code_bytes(4, 256, 0) == 0
    assert L.sg_kv8_code_bytes(4, 256, 1) == 16 * 4 * 512
    assert L.sg_kv8_code_bytes(4, 256, 262144) == 262144 * 4 * 512
    assert L.sg_kv8_code_bytes(8, 128, (1 << 32) - 1) == (1 << 32) * 8 * 256         # past 32 bits
    assert L.sg_kv8_scale_bytes(4, 32, 33) == 2 * 4 * 8
    assert L.sg_kv8_code_bytes(4, 96, 16) == 0 and L.sg_kv8_scale_bytes(4, 48, 16) == 0 and L.sg_kv8_code_bytes(0, 64, 16) == 0
    assert L.sg_kv8_code_bytes(4, 64, 1 << 32) == 0


@pytest.mark.parametrize("name", ["sg_gpu_run_kv8_store", "sg_gpu_run_kv8_load"])
@pytest.mark.parametrize("change,match", [
    ({0: 0}, "n_kv"), ({1: 96}, "head_dim"), ({1: 0}, "head_dim"), ({2: 8}, "block"), ({2: 48}, "block"),
    ({3: 65}, "codes"), ({3: 0xFFFFFFF0}, "positions"), ({4: 0}, "n must"), ({4: 1 << 28}, "codes"), ({5: 255}, "stride"),
    ({4: 60, 5: 1000}, "k holds"), ({4: 0xFFFFFFFF}, "positions")])
def test_store_and_load_refuse(name, change, match):
    # 2 kv heads x 128, block 16, 68 positions' room; rows [4, 4 + 60) of 256 floats
    p = [2, 128, 16, 4, 60, 0]
    for i, v in change.items():
        p[i] = v
    k, v, codes, scales = far(60 * 256 * 4), far(60 * 256 * 4), far(5 * 2 * 32 * 128), far(5 * 2 * 8)
    h = (k, v, codes, scales) if name.endswith("store") else (codes, scales, k, v)
    refused(name, h, p, match)


def test_store_and_load_refuse_short_misaligned_and_overlapping_buffers():
    p, rb, cb, sb = [2, 128, 16, 0, 20, 0], 20 * 256 * 4, 2 * 2 * 32 * 128, 2 * 2 * 8
    k, v, c, s = far(rb), far(rb), far(cb), far(sb)
    st, ld = "sg_gpu_run_kv8_store", "sg_gpu_run_kv8_load"
    refused(st, (far(rb - 4), v, c, s), p, "k holds")
    refused(st, (k, far(rb - 4), c, s), p, "v holds")
    refused(st, (k, v, far(cb - 1), s), p, "codes holds")
    refused(st, (k, v, c, far(sb - 1)), p, "scales holds")
    refused(st, (k, v, buf(cb, AT + 8), s), p, "aligned")
    refused(st, (k, v, c, buf(sb, AT + 2)), p, "aligned")
    refused(st, (buf(rb, AT + 1), v, c, s), p, "aligned")
    refused(st, (k, v, buf(cb), buf(sb, AT + cb - 4)), p, "overlap")
    refused(st, (buf(rb, AT + 16), v, buf(cb), s), p, "overlap")
    refused(ld, (c, s, buf(rb), buf(rb, AT + rb - 4)), p, "overlap")
    refused(ld, (c, s, k, k), p, "overlap")
    # rows of one allocation that would collide at this stride
    p[5] = 500
    n = (19 * 500 + 256) * 4
    refused(ld, (c, s, buf(n), buf(n, AT + 250 * 4)), p, "overlap")
    for i in range(4):
        h = [k, v, c, s]
        h[i] = None
        refused(st, h, p, "NULL")
    refused(st, (k, v, c, s), None, "NULL")


@pytest.mark.parametrize("change,match", [
    ({0: 0}, "n_heads"), ({0: 5}, "n_heads"), ({0: 34}, "n_heads"), ({1: 0}, "n_kv"), ({2: 32}, "head_dim"), ({3: 97}, "codes"),
    ({4: 63}, "q_stride"), ({4: 1 << 20}, "q holds"), ({6: 24}, "block"), ({3: 0xFFFFFFFF}, "positions")])
def test_attn_decode_refuses(change, match):
    p = [4, 2, 64, 96, 64, F(0.125), 32]
    for i, v in change.items():
        p[i] = v
    refused("sg_gpu_run_attn_decode_kv8", (far(34 * 64 * 4), far(6 * 2 * 32 * 64), far(3 * 2 * 8), far(34 * 64 * 4)), p, match)


@pytest.mark.parametrize("change,match", [
    ({0: 5}, "n_heads"), ({4: 0}, "n is zero"), ({3: 91}, "codes"), ({3: 0xFFFFFFFF, 4: 2}, "positions"),
    ({4: 7}, "q holds"), ({7: 0}, "block"), ({5: 60}, "q_stride")])
def test_attn_prefill_refuses(change, match):
    p = [4, 2, 64, 90, 6, 64, F(0.125), 32]
    for i, v in change.items():
        p[i] = v
    n = 6 * 4 * 64 * 4
    refused("sg_gpu_run_attn_prefill_kv8", (far(n), far(7 * 2 * 32 * 64 if 7 in change or 4 in change else 6 * 2 * 32 * 64),
                                            far(6 * 4 * 8), far(n)), p, match)


def test_attn_refuses_overlap_and_null():
    p = [4, 2, 64, 96, 64, F(0.125), 32]
    q, c, s, o = far(1024), far(6 * 2 * 32 * 64), far(3 * 2 * 8), far(1024)
    f = "sg_gpu_run_attn_decode_kv8"
    refused(f, (q, c, s, q), p, "overlap")
    refused(f, (q, buf(6 * 2 * 32 * 64), s, buf(1024, AT + 1024)), p, "overlap")
    refused(f, (q, c, s, buf(1024, AT + 2)), p, "aligned")
    refused(f, (q, c, s, None), p, "NULL")
    refused(f, (q, c, s, o), None, "NULL")
    refused("sg_gpu_run_attn_prefill_kv8", (q, c, s, o), None, "NULL")


@pytest.mark.parametrize("change,match", [
    ({0: 0}, "shape"), ({0: 257}, "shape"), ({1: 0}, "shape"), ({1: 65}, "shape"), ({1: 31}, "shape"), ({2: 0}, "shape"),
    ({3: 63}, "shape"), ({4: 0}, "shape"), ({5: 6 | 5 << 8 | 4 << 16}, "sections"), ({5: 6 | 5 << 8 | 5 << 16 | 2 << 24}, "sections"),
    ({5: 0 | 16 << 8 | 0 << 16 | 1 << 24}, "interleaved"), ({5: 10 | 0 << 8 | 6 << 16 | 1 << 24}, "interleaved"), ({6: F(0.0)}, "theta"),
    ({6: F(math.inf)}, "theta"), ({6: F(math.nan)}, "theta"), ({7: 127}, "row stride"), ({4: 11}, "x holds"), ({7: 4000}, "x holds")])
def test_rope_axes_refuses(change, match):
    p = [64, 32, 2, 0, 10, 6 | 5 << 8 | 5 << 16, F(1e7), 0]
    for i, v in change.items():
        p[i] = v
    refused("sg_gpu_run_rope_axes", (far(10 * 128 * 4), far(10 * 12), far(10 * 128 * 4)), p, match)


def test_sizes_that_wrap_64_bits_are_refused():
    """Strides whose product with the row count passes 2^64 must not come out small."""
    big = 0xFFFFFFFF
    refused("sg_gpu_run_rope_axes", (far(1 << 20), far(1 << 40), far(1 << 20)),
            [64, 32, 65535, big - 3, big, 6 | 5 << 8 | 5 << 16, F(1e7), 0], "too large")
    refused("sg_gpu_run_attn_prefill_kv8", (far(1 << 20), far(1 << 62), far(1 << 62), far(1 << 20)),
            [65535 * 16, 65535, 64, 0, 1 << 26, big, F(0.1), 128], "too large")
    refused("sg_gpu_run_attn_prefill_kv8", (far(1 << 20), far(1 << 62), far(1 << 62), far(1 << 20)),
            [16, 1, 64, 0, (1 << 26) + 1, 64, F(0.1), 128], "2\\^30")
    assert S.lib().sg_kv8_code_bytes(65536, 256, 1 << 31) == 0 and S.lib().sg_kv8_scale_bytes(1 << 20, 16, 1 << 31) == 0


def test_rope_axes_refuses_overlap():
    p = [64, 32, 2, 0, 10, 6 | 5 << 8 | 5 << 16, F(1e7), 0]
    n = 10 * 128 * 4
    refused("sg_gpu_run_rope_axes", (buf(n), far(120), buf(n, AT + 4)), p, "overlap")
    refused("sg_gpu_run_rope_axes", (far(n), buf(120), buf(n, AT + 64)), p, "overlap")
    refused("sg_gpu_run_rope_axes", (far(n), far(119), far(n)), p, "pos holds")


@pytest.mark.parametrize("p,match", [([4, 0, 1, 0], "shape"), ([4, 100, 0, 0], "shape"), ([4, 100, 70000, 0], "shape"),
                                     ([4, 100, 1, 2], "shape"), ([4, 101, 1, 0], "counts holds"), ([5, 100, 1, 0], "ids holds"),
                                     ([4, 1 << 31, 1, 0], "shape")])
def test_token_counts_refuses(p, match):
    refused("sg_gpu_run_token_counts", (far(16), far(400)), p, match)
    c = buf(400)
    refused("sg_gpu_run_token_counts", (buf(16, AT + 396), c), [4, 100, 1, 0], "overlap")
    refused("sg_gpu_run_token_counts", (None, c), [4, 100, 1, 0], "NULL")


@pytest.mark.parametrize("change,match", [
    ({0: 0}, "shape"), ({0: 1 << 31}, "shape"), ({1: 0}, "shape"), ({1: 65536}, "shape"), ({2: F(0.0)}, "repetition"),
    ({2: F(-1.0)}, "repetition"), ({2: F(math.nan)}, "repetition"), ({2: F(math.inf)}, "repetition"), ({3: F(math.nan)}, "frequency"),
    ({4: F(math.inf)}, "presence"), ({0: 101}, "logits holds"), ({1: 3}, "logits holds")])
def test_logits_refuses(change, match):
    p = [100, 2, F(1.1), F(0.1), F(0.2)]
    for i, v in change.items():
        p[i] = v
    h = [far(800), far(800), far(400), far(32), far(800), far(8)]
    refused("sg_gpu_run_logits", h, p, match)


def test_logits_refuses_short_and_overlapping_buffers():
    p = [100, 2, F(1.1), F(0.1), F(0.2)]
    sizes, names = [800, 800, 400, 32, 800, 8], ["logits", "counts", "bias", "mask", "out", "token"]
    for i, n in enumerate(names):
        h = [far(x) for x in sizes]
        h[i] = far(sizes[i] - 1)
        refused("sg_gpu_run_logits", h, p, n + " holds")
        h[i] = buf(sizes[i], AT + 2)
        refused("sg_gpu_run_logits", h, p, "aligned")
        if n in ("logits", "out", "token"):
            h[i] = None
            refused("sg_gpu_run_logits", h, p, "NULL")
    for i in range(5):
        h = [far(x) for x in sizes]
        h[i], h[5] = buf(sizes[i]), buf(8, AT)
        refused("sg_gpu_run_logits", h, p, "overlap")
    for i, at in ((0, AT + 4), (1, AT), (2, AT), (3, AT)):
        h = [far(x) for x in sizes]
        h[i], h[4] = buf(sizes[i]), buf(800, at)
        refused("sg_gpu_run_logits", h, p, "overlap")


def test_oracle_store_rows_one_by_one_or_together():
    """The oracle's own check: stored values are within half a step (and half a step more per
    growth of the scale) of the rows."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 40, 2, 64)).astype(np.float32)
    a, b = K.Cache(2, 64, 32, 40), K.Cache(2, 64, 32, 40)
    a.store(x[0], x[1], 0)
    for i in range(40):
        b.store(x[0, i:i + 1], x[1, i:i + 1], i)
    for half in range(2):
        step = a.scales[np.arange(40) // 32, :, half][:, :, None]
        assert np.array_equal(a.scales, b.scales)
        assert (np.abs(a.values(half, 40) - x[half]) <= 0.5001 * step).all()
        assert (np.abs(b.values(half, 40) - x[half]) <= 0.5001 * step * 8).all()


@pytest.mark.parametrize("make", [list, tuple, iter, lambda v: (x for x in v), lambda v: map(int, v), lambda v: dict.fromkeys(v).keys(),
                                  lambda v: np.array(v, np.int64)])
def test_params_takes_what_can_be_iterated(make):
    """Whatever holds the values, and values that are not unsigned 32-bit integers: low 32 bits of each, zeros behind."""
    assert list(S.params(make([1, 2, 3]))) == [1, 2, 3, 0, 0, 0, 0, 0]
    assert list(S.params(make([5, -1, 1 << 33 | 7]))) == [5, 0xFFFFFFFF, 7, 0, 0, 0, 0, 0]
    assert list(S.params(make([]))) == [0] * 8
    assert list(S.params(make(range(8)))) == list(range(8))
    with pytest.raises(IndexError):
        S.params(make(range(9)))


def test_params_of_floats():
    assert list(S.params(x for x in (1.0, np.float32(2.5), np.int32(-2)))) == [1, 2, 0xFFFFFFFE, 0, 0, 0, 0, 0]


def test_attention_parts():
    """The query of how attention over the 8-bit cache runs: on the host alone, 0 for what a call would refuse."""
    def parts(*a):
        w = C.c_uint32(9)
        return S.lib().sg_gpu_attn_kv8_parts(G, *a, C.byref(w)), w.value
    assert parts(24, 4, 256, 17003, 1) == (64, 4) and parts(24, 4, 256, 383, 1) == (1, 8) and parts(24, 4, 256, 14336, 2048)[1] == 0
    assert S.lib().sg_gpu_attn_kv8_parts(G, 24, 4, 256, 17003, 1, None) == 64
    assert S.lib().sg_gpu_attn_kv8_parts(None, 24, 4, 256, 17003, 1, None) == 0
    for bad in ((24, 4, 256, 17003, 0), (24, 5, 256, 0, 1), (0, 4, 256, 0, 1), (24, 0, 256, 0, 1), (17, 1, 64, 0, 1), (24, 4, 96, 0, 1),
                (65536, 65536, 64, 0, 1), (24, 4, 256, 0xFFFFFFFF, 1), (16, 1, 64, 0, (1 << 26) + 1)):
        assert parts(*bad) == (0, 0)
