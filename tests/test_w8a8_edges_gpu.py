"""INT8 x INT8 products: weights quantised on the device right ahead of the product that reads them."""
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
