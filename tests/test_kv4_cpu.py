"""What the 4-bit cache calls refuse, before anything is launched. The calls read and write only the error fields of the context then,
so a zeroed one stands in for it and no GPU is needed."""
import ctypes as C

import pytest

from libinferbit_b200 import Kv4T, _ffi

lib = _ffi.load_ibcu()
pytestmark = pytest.mark.skipif(lib.ibcu_device_count() > 0, reason="with a GPU, a call that is not refused would launch")
P = 1 << 20                                       # an aligned address that nothing reads


def refused(call, *args):
    ctx = C.create_string_buffer(1 << 16)
    rc = call(ctx, *args)
    return rc == -1 and len(lib.ibcu_last_error(ctx)) > 0


def cache(**kw):
    f = {"k": P, "v": 2 * P, "scale": 3 * P, "weight": None, "decay": 1.0, "n_kv_heads": 2, "head_dim": 64, "max_rows": 64, **kw}
    return C.pointer(Kv4T(*(f[n] for n, _ in Kv4T._fields_)))


BAD_CACHES = [dict(k=None), dict(v=None), dict(scale=None), dict(k=P + 8), dict(v=P + 4), dict(scale=P + 2), dict(weight=P + 2), dict(head_dim=0), dict(head_dim=80), dict(head_dim=16),
              dict(head_dim=512), dict(head_dim=-32), dict(n_kv_heads=0), dict(n_kv_heads=-1), dict(max_rows=0), dict(max_rows=63), dict(max_rows=-8),
              dict(weight=P, decay=-0.5), dict(weight=P, decay=1.5), dict(weight=P, decay=float("nan"))]


@pytest.mark.parametrize("bad", BAD_CACHES, ids=lambda b: ",".join(f"{k}={v}" for k, v in b.items()))
def test_caches(bad):
    t, good = cache(**bad), cache(weight=P)
    assert refused(lib.ibcu_kv4_write, t, P, P, 0, 0, 1, 10000.0)
    assert refused(lib.ibcu_kv4_read, t, P, P, 0, 1)
    assert refused(lib.ibcu_attention_kv4, t, P, P, 4, 0, 1)
    assert refused(lib.ibcu_attention_decode_kv4, t, P, P, P, P, 4, 0, 0, 1, 10000.0)
    assert refused(lib.ibcu_attention_decode_kv4_at, t, P, P, P, P, 4, P, 1, 10000.0)
    assert refused(lib.ibcu_kv4_evict, t, good, 8, 4, 0, 0, None) and refused(lib.ibcu_kv4_evict, good, t, 8, 4, 0, 0, None)


def test_no_cache_and_no_context():
    assert refused(lib.ibcu_kv4_write, None, P, P, 0, 0, 1, 0.0)
    assert lib.ibcu_kv4_write(None, cache(), P, P, 0, 0, 1, 0.0) == -1
    assert lib.ibcu_kv4_evict(None, cache(), cache(), 8, 4, 0, 0, None) == -1


@pytest.mark.parametrize("row0,B", [(-1, 1), (64, 1), (60, 5), (0, 0), (0, -3), (2**31 - 1, 2**31 - 1)])
def test_rows(row0, B):
    t = cache()
    assert refused(lib.ibcu_kv4_write, t, P, P, row0, 0, B, 0.0)
    assert refused(lib.ibcu_kv4_read, t, P, P, row0, B)
    assert refused(lib.ibcu_attention_kv4, t, P, P, 4, row0, B)
    assert refused(lib.ibcu_attention_decode_kv4, t, P, P, P, P, 4, row0, 0, B, 0.0)


@pytest.mark.parametrize("pos0,theta", [(-1, 10000.0), (2**31 - 1, 10000.0), (0, -1.0), (0, float("nan")), (0, float("inf"))])
def test_rotations(pos0, theta):
    assert refused(lib.ibcu_kv4_write, cache(), P, P, 0, pos0, 2, theta)
    assert refused(lib.ibcu_attention_decode_kv4, cache(), P, P, P, P, 4, 0, pos0, 2, theta)


@pytest.mark.parametrize("heads", [0, -2, 3, 1])
def test_heads(heads):
    assert refused(lib.ibcu_attention_kv4, cache(), P, P, heads, 0, 1)
    assert refused(lib.ibcu_attention_decode_kv4, cache(), P, P, P, P, heads, 0, 0, 1, 0.0)


@pytest.mark.parametrize("at", range(2))
def test_null_vectors(at):
    two = [P, P]; two[at] = None
    assert refused(lib.ibcu_kv4_write, cache(), *two, 0, 0, 1, 0.0) and refused(lib.ibcu_kv4_read, cache(), *two, 0, 1)
    assert refused(lib.ibcu_attention_kv4, cache(), *two, 4, 0, 1)
    for i in range(4):
        four = [P] * 4; four[i] = None
        assert refused(lib.ibcu_attention_decode_kv4, cache(), *four, 4, 0, 0, 1, 0.0)


@pytest.mark.parametrize("rows,keep,sink,recent", [(0, 0, 0, 0), (65, 4, 0, 0), (8, 9, 0, 0), (8, 0, 0, 0), (8, 4, -1, 0), (8, 4, 0, -1), (8, 4, 3, 2), (8, 4, 2**31 - 1, 2**31 - 1), (64, 20, 0, 0)])
def test_evictions(rows, keep, sink, recent):
    assert refused(lib.ibcu_kv4_evict, cache(weight=P), cache(weight=P, max_rows=16), rows, keep, sink, recent, None)


def test_evictions_between_unlike_caches():
    assert refused(lib.ibcu_kv4_evict, cache(), cache(weight=P), 8, 4, 0, 0, None)                    # no weights to go by
    assert refused(lib.ibcu_kv4_evict, cache(weight=P), cache(n_kv_heads=1), 8, 4, 0, 0, None)
    assert refused(lib.ibcu_kv4_evict, cache(weight=P), cache(head_dim=32), 8, 4, 0, 0, None)


def test_evictions_into_a_cache_that_shares_some_planes():
    assert refused(lib.ibcu_kv4_evict, cache(weight=P), cache(weight=P, k=8 * P), 8, 4, 0, 0, None)
    assert refused(lib.ibcu_kv4_evict, cache(weight=P), cache(weight=P, max_rows=32), 8, 4, 0, 0, None)


@pytest.mark.parametrize("heads,at,B,theta", [(4, None, 1, 1.0), (4, P, 65, 1.0), (4, P, 0, 1.0), (3, P, 1, 1.0), (4, P, 1, -1.0)])
def test_places_on_the_device(heads, at, B, theta):
    assert refused(lib.ibcu_attention_decode_kv4_at, cache(), P, P, P, P, heads, at, B, theta)
