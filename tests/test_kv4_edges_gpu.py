"""The 4-bit KV cache where it can go wrong: groups that hold NaN, in every form of the attention."""
import numpy as np
import pytest

from tests import _kv4
from tests.test_kv4_gpu import _free, get, put  # noqa: F401

pytestmark = pytest.mark.gpu

# tiles of 4, 8 and 16 columns, and of 128 for heads of 128 and 64
FORMS = [(8, 2, 64, 700, 1), (32, 8, 128, 90, 1), (16, 2, 128, 700, 1), (8, 2, 96, 500, 30), (12, 4, 64, 40, 60), (8, 2, 128, 300, 700), (32, 8, 128, 200, 250), (8, 2, 64, 300, 1000)]


def step(be, planes, q, n_heads, row0):
    B, R = q.shape[0], row0 + q.shape[0]
    t, o = put(be, *planes, weight=np.zeros(planes[0].shape[:2]), decay=0.0), be.alloc(q.nbytes)
    dq = be.upload(q)
    be._check(be.lib.ibcu_attention_kv4(be.ctx, t, dq.ptr, o.ptr, n_heads, row0, B)); be.sync()
    return be.download(o, np.float32, q.size).reshape(B, n_heads, -1, 32), get(be, t)[3][:, :R]


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", FORMS)
def test_a_value_group_with_nan_spoils_its_own_outputs(backend, n_heads, n_kv, hd, row0, B):
    """NaN in one value group of two rows of one KV head: the group's outputs of that head's queries from the first such position on, nothing else; no weight."""
    be, rng = backend, np.random.default_rng(n_heads + hd + B)
    R, ng = row0 + B, hd // 32
    planes = _kv4.random_planes(rng, n_kv, hd, (R + 7) // 8 * 8, R)
    q = rng.standard_normal((B, n_heads * hd), dtype=np.float32)
    want, weight, tol, wtol = _kv4.attention(q.astype(np.float64), _kv4.plane_values(*(p[:, :R] for p in planes)), n_heads, row0)
    want, tol = want.reshape(B, n_heads, ng, 32), tol.reshape(B, n_heads, ng, 32)
    head, group, first = n_kv - 1, ng - 1, row0 + B // 3
    for at in (first, min(R - 1, first + 70)):
        planes[2][head, at, ng + group] = np.nan
    got, drawn = step(be, planes, q, n_heads, row0)
    spoilt = np.zeros(got.shape, bool)
    spoilt[first - row0:, head * (n_heads // n_kv):, group] = True
    assert np.array_equal(np.isnan(got), spoilt)
    assert np.all(np.abs(got - want)[~spoilt] <= tol[~spoilt])
    assert np.all(np.abs(drawn - weight) <= wtol + 2.0 ** -24 * weight)


@pytest.mark.parametrize("n_heads,n_kv,hd,row0,B", FORMS)
def test_a_key_group_with_nan_spoils_what_sees_it(backend, n_heads, n_kv, hd, row0, B):
    """NaN in a key group of one KV head: all outputs of that head's queries from its position on and the weights of all rows that these see; the other heads keep theirs."""
    be, rng = backend, np.random.default_rng(n_heads + hd + B + 1)
    R, ng, per = row0 + B, hd // 32, n_heads // n_kv
    planes = _kv4.random_planes(rng, n_kv, hd, (R + 7) // 8 * 8, R)
    q = rng.standard_normal((B, n_heads * hd), dtype=np.float32)
    want, weight, tol, wtol = _kv4.attention(q.astype(np.float64), _kv4.plane_values(*(p[:, :R] for p in planes)), n_heads, row0)
    want, tol = want.reshape(B, n_heads, ng, 32), tol.reshape(B, n_heads, ng, 32)
    at = row0 + B // 3
    planes[2][0, at, 0] = np.nan
    got, drawn = step(be, planes, q, n_heads, row0)
    spoilt = np.zeros(got.shape, bool)
    spoilt[at - row0:, :per] = True
    assert np.array_equal(np.isnan(got), spoilt)
    assert np.all(np.abs(got - want)[~spoilt] <= tol[~spoilt])
    assert np.isnan(drawn[0]).all() and np.all(np.abs(drawn[1:] - weight[1:]) <= wtol[1:] + 2.0 ** -24 * weight[1:])


@pytest.mark.parametrize("n_heads,n_kv,hd,B", [(8, 2, 64, 2), (8, 2, 64, 40), (8, 8, 128, 700)])
def test_positions_at_the_end_of_31_bits(backend, n_heads, n_kv, hd, B):
    """The last positions there are give what the call with arguments gives; further ones, read from the device, write nothing and are reported."""
    be, rng = backend, np.random.default_rng(B)
    max_rows, theta = (B + 8) // 8 * 8, 500000.0
    planes = _kv4.random_planes(rng, n_kv, hd, max_rows, max_rows)
    x = [rng.standard_normal((B, heads * hd), dtype=np.float32) for heads in (n_heads, n_kv, n_kv)]
    d = [be.upload(a) for a in x]
    last, at, outs = 2**31 - 1 - B, be.upload(np.zeros(2, np.int32)), []
    for device in (False, True):
        t, o = put(be, *planes), be.alloc(B * n_heads * hd * 4)
        be.write(at, np.array([0, last], np.int32))
        if device:
            be._check(be.lib.ibcu_attention_decode_kv4_at(be.ctx, t, *(a.ptr for a in d), o.ptr, n_heads, at.ptr, B, theta))
        else:
            be._check(be.lib.ibcu_attention_decode_kv4(be.ctx, t, *(a.ptr for a in d), o.ptr, n_heads, 0, last, B, theta))
        be.sync()
        outs.append((be.download(o, np.float32, B * n_heads * hd).reshape(B, -1), *(a.tobytes() for a in get(be, t))))
    assert outs[0][1:] == outs[1][1:]
    tol = _kv4.attention(_kv4.rotate(x[0], n_heads, last, theta), _kv4.plane_values(*(a[:, :B] for a in get(be, t))), n_heads, 0)[2]
    assert np.all(np.abs(outs[0][0] - outs[1][0]) <= 2 * tol)         # each is within it of the sums in 64 bits
    assert be.lib.ibcu_attention_decode_kv4(be.ctx, t, *(a.ptr for a in d), o.ptr, n_heads, 0, last + 1, B, theta) == -1
    be.lib.ibcu_clear_error(be.ctx)
    for pos in (last + 1, 2**31 - 1):
        before = [a.tobytes() for a in get(be, t)]
        be.write(at, np.array([0, pos], np.int32))
        be._check(be.lib.ibcu_attention_decode_kv4_at(be.ctx, t, *(a.ptr for a in d), o.ptr, n_heads, at.ptr, B, theta))
        assert be.lib.ibcu_sync(be.ctx) == -1 and b"outside the cache" in be.lib.ibcu_last_error(be.ctx)
        be.lib.ibcu_clear_error(be.ctx)
        assert [a.tobytes() for a in get(be, t)] == before
