"""INT8 x INT8 products at their edges: weights quantised on the device right ahead of the product that reads them, the largest sums."""
import numpy as np
import pytest

from libinferbit_b200 import LinearT
from tests import test_w8a8_gpu as base
from tests.test_w8a8_gpu import _free  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,B,form", [(300, 4096, 1, "codes"), (300, 4096, 1, "fp32"), (300, 4096, 2, "linear"), (300, 4096, 24, "codes"), (300, 4096, 24, "fp32"),
                                        (4096, 512, 1, "fp32"), (2600, 4096, 600, "codes"), (2600, 4096, 600, "fp32"), (300, 4096, 24, "linear")])
def test_weights_quantised_right_before_the_product(backend, M, N, B, form):
    """Fresh weights into the same tensor again and again, no waiting between the quantiser and the product (a warp a row, tiles, pairs of blocks, ibcu_linear): the bits of the same
    calls with a wait between them."""
    be, rng = backend, np.random.default_rng(M + B)
    sets = [be.upload(rng.standard_normal((M, N), dtype=np.float32) * np.float32(0.1 + i)) for i in range(4)]
    x = rng.standard_normal((B, N), dtype=np.float32)
    q, sx = base.quantise(x)
    dx, dq, ds, w, sw = be.upload(x), be.upload(q), be.upload(sx), be.alloc(M * N), be.alloc(M * 4)
    rounds = 24

    def run(wait):
        outs = [be.alloc(B * M * 4) for _ in range(rounds)]
        for i, o in enumerate(outs):
            t = (LinearT * 1)(LinearT(w.ptr, sw.ptr, o.ptr, M, M, 1, 0))
            be._check(be.lib.ibcu_quantize_rows_int8(be.ctx, sets[i * 7 % 4].ptr, w.ptr, sw.ptr, N, M))
            if wait:
                be.sync()
            if form == "codes":
                be._check(be.lib.ibcu_linear_w8a8(be.ctx, t, 1, dq.ptr, ds.ptr, N, B))
            elif form == "fp32":
                be._check(be.lib.ibcu_linear_w8a8_fp32(be.ctx, t, 1, dx.ptr, N, B))
            else:
                be._check(be.lib.ibcu_linear(be.ctx, t, 1, dx.ptr, N, B, 8))
            if wait:
                be.sync()
        be.sync()
        return [be.download(o, np.float32, B * M) for o in outs]

    want = run(True)
    assert not np.array_equal(want[0], want[1])
    for a, b in zip(want, run(False)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("M,B", [(40, 1), (300, 9), (9700, 5), (9700, 300)])
@pytest.mark.parametrize("add", [0, 1])
def test_the_largest_sums_of_any_codes(backend, M, B, add):
    """131072 columns of -128 by -128 are 2^31, one more than an int32 holds; beside it the largest and smallest sums of the other codes. Scales of 1: every sum is a float."""
    be, N = backend, 131072
    w, x = be.alloc(M * N), be.alloc(B * N)
    sw, sx, o = be.upload(np.ones(M, np.float32)), be.upload(np.ones(B, np.float32)), be.alloc(B * M * 4)
    t = (LinearT * 1)(LinearT(w.ptr, sw.ptr, o.ptr, M, M, 1, add))
    for a, b in ((-128, -128), (-128, 127), (127, -128), (-127, -128), (-128, -127), (127, 127)):
        be._check(be.lib.ibcu_memset(be.ctx, w.ptr, a & 255, M * N)); be._check(be.lib.ibcu_memset(be.ctx, x.ptr, b & 255, B * N)); be._check(be.lib.ibcu_memset(be.ctx, o.ptr, 0, B * M * 4))
        be._check(be.lib.ibcu_linear_w8a8(be.ctx, t, 1, x.ptr, sx.ptr, N, B)); be.sync()
        assert np.all(be.download(o, np.float32, B * M) == np.float32(a * b * N)), (a, b)
    # one code less in the first token: 128 below 2^31, the float next to it
    be.write(x, np.array([-127], np.int8)); be._check(be.lib.ibcu_memset(be.ctx, w.ptr, 128, M * N))
    be._check(be.lib.ibcu_memset(be.ctx, x.at(1), 128, B * N - 1)); be._check(be.lib.ibcu_memset(be.ctx, o.ptr, 0, B * M * 4))
    be._check(be.lib.ibcu_linear_w8a8(be.ctx, t, 1, x.ptr, sx.ptr, N, B)); be.sync()
    got = be.download(o, np.float32, B * M).reshape(B, M)
    assert np.all(got[0] == np.float32(2.0 ** 31 - 128)) and np.all(got[1:] == np.float32(2.0 ** 31))
