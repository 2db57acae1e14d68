"""How far attention over the 4-bit cache is off 64 bits, form by form, against what each form's own additions may lose.

The tensor cores cut every addition off towards zero: half a step of 2^-23 to 2^-24 of the sum on the mean, 0.36 * 2^-23, of a partial sum that has grown to sqrt(t / T) of the
whole after t of T additions: 0.24 T * 2^-23 of the result, all towards zero, so that adding up more such sums does not average it out.
  mma.sync: 32 rows are a sum (2 additions, 4 in tiles of 16 columns) and so is a group of 32 products of a score (as many): 1.1e-7 each. Queries and weights in two pieces
  (2^-22 left out, a third of that on the mean), the approximate exponential, the groups' and the partial sums' FP32 additions: 1e-7 each. Together, as independent
  errors, 2.5e-7, and half of that again for what is not independent. Without the sums of 32 rows, 16000 rows would be off by ten times as much.
  tcgen05: 192 rows are a sum of 36 additions, a score one of 24: 1.03e-6 and 0.69e-6 (scores are of size 1), together 1.24e-6. One sum for 2048 rows was 2.3e-6 off, for 16000
  5.7e-5."""
import numpy as np
import pytest

from tests import _kv4
from tests.test_kv4_gpu import _free, put  # noqa: F401

pytestmark = pytest.mark.gpu
MMA_SYNC, TCGEN05 = 1.5 * 2.5e-7, 1.24e-6


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B,bound", [(8, 1, 128, 30000, 1, MMA_SYNC), (4, 1, 64, 30000, 1, MMA_SYNC), (32, 8, 128, 12000, 2, MMA_SYNC), (8, 2, 128, 12000, 60, MMA_SYNC),
                                                          (4, 1, 96, 12000, 100, MMA_SYNC), (2, 1, 256, 16000, 30, MMA_SYNC), (8, 1, 128, 8000, 640, TCGEN05), (8, 1, 64, 8000, 900, TCGEN05),
                                                          (32, 8, 128, 0, 1500, TCGEN05)])
def test_off_64_bits(backend, n_heads, n_kv, hd, row0, B, bound):
    be, rng = backend, np.random.default_rng(row0 + hd)
    R, per = row0 + B, n_heads // n_kv
    planes = _kv4.random_planes(rng, n_kv, hd, (R + 7) // 8 * 8, R)
    q = rng.standard_normal((B, n_heads, hd), dtype=np.float32)
    dq, do = be.upload(q), be.alloc(q.nbytes)
    be._check(be.lib.ibcu_attention_kv4(be.ctx, put(be, *planes), dq.ptr, do.ptr, n_heads, row0, B)); be.sync()
    got = be.download(do, np.float32, q.size).reshape(q.shape)
    K, V = _kv4.plane_values(*(p[:, :R] for p in planes))
    off = size = 0.0
    for h in range(0, n_heads, max(1, n_heads // 8)):
        s = q[:, h].astype(np.float64) @ K[h // per].T / np.sqrt(hd)
        p = np.where(np.arange(R)[None] <= row0 + np.arange(B)[:, None], np.exp(s - s.max(1, keepdims=True)), 0.0)
        want = p @ V[h // per] / p.sum(1, keepdims=True)
        off, size = off + ((got[:, h] - want) ** 2).sum(), size + (want ** 2).sum()
    print(f"{np.sqrt(off / size):.2e} of {bound:.2e}")
    assert np.sqrt(off / size) <= bound, np.sqrt(off / size)
