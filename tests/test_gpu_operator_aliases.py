"""In place through another handle of the same device memory: the rotary axes
and the logits take their input's data, whichever of the two handles has a host
mirror, and what lies behind either stays (include/surge.h)."""
import ctypes as C

import numpy as np
import pytest

import surge_amd as S
from test_gpu_kv8 import Bufs

pytestmark = pytest.mark.gpu
F = S.fbits


class Alias:
    """A handle of the device memory of buf's first `nbytes`, without a mirror."""

    def __init__(self, gpu, buf, nbytes):
        self.handle = C.c_void_p()
        S.check(S.lib().sg_gpu_wrap_device(gpu.handle, S.lib().sg_gpu_buf_device(buf.handle), nbytes, C.byref(self.handle)))

    def free(self):
        S.lib().sg_gpu_buf_free(self.handle)


def calls(rng):
    """(input [n] f32, call(gpu, buf, in, out)) of each operator that may work in place."""
    n, nh, hd = 3, 2, 64
    pos = rng.integers(0, 5000, (3, n)).astype(np.int32)

    def rope(gpu, buf, x, out):
        gpu.rope_axes(x, buf(pos), out, [hd, 32, nh, 0, n, 6 | 5 << 8 | 5 << 16, F(1e7), 0])

    def logits(gpu, buf, x, out):
        tok = buf(np.zeros(n, np.uint32))
        gpu.logits(x, buf(np.ones((n, nh * hd), np.uint32)), None, None, out, tok, [nh * hd, n, F(1.5), F(0.25), F(0.1)])

    return (rng.standard_normal(n * nh * hd).astype(np.float32), rope), (rng.standard_normal(n * nh * hd).astype(np.float32), logits)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("tail", [0, 5])
@pytest.mark.parametrize("cover", ["call", "all"])
def test_input_is_an_alias_of_the_output(gpu, which, tail, cover):
    """The output has a mirror with something else in it; the data are on the device alone."""
    x, call = calls(np.random.default_rng(which))[which]
    with Bufs(gpu) as buf:
        want = buf(np.zeros_like(x))
        call(gpu, buf, buf(x), want)
        on_device = np.concatenate([x, np.full(tail, 3.0, np.float32)])
        out = buf(on_device)
        S.check(S.lib().sg_gpu_buf_upload(out.handle))
        out.array[...] = 7.0
        a = Alias(gpu, out, x.nbytes if cover == "call" else out.nbytes)
        call(gpu, buf, a, out)
        assert np.array_equal(out.array[:x.size], want.array)
        # behind the call: the input's data where the input reaches, else the output's own
        assert (out.array[x.size:] == (7.0 if cover == "call" else 3.0)).all()
        a.free()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("tail", [0, 5])
def test_output_is_an_alias_of_the_input(gpu, which, tail):
    """The input has the mirror: it holds the result afterwards, and a second call goes on from that."""
    x, call = calls(np.random.default_rng(which))[which]
    with Bufs(gpu) as buf:
        once, twice = buf(np.zeros_like(x)), buf(np.zeros_like(x))
        call(gpu, buf, buf(x), once)
        call(gpu, buf, buf(once.array.copy()), twice)
        src = buf(np.concatenate([x, np.full(tail, 3.0, np.float32)]))
        a = Alias(gpu, src, src.nbytes)
        for want in (once, twice):
            call(gpu, buf, src, a)
            assert np.array_equal(src.array[:x.size], want.array) and (src.array[x.size:] == 3.0).all()
        a.free()
