"""What the INT8 x INT8 calls refuse before anything is launched (see test_kv4_cpu.py for the zeroed context)."""
import ctypes as C

import pytest

from libinferbit_b200 import LinearT, _ffi

lib = _ffi.load_ibcu()
pytestmark = pytest.mark.skipif(lib.ibcu_device_count() > 0, reason="with a GPU, a call that is not refused would launch")
P = 1 << 20


def refused(call, *args):
    ctx = C.create_string_buffer(1 << 16)
    return call(ctx, *args) == -1 and len(lib.ibcu_last_error(ctx)) > 0


def tensor(**kw):
    f = {"w": P, "scales": P, "out": P, "M": 64, "out_stride": 64, "scales_fp32": 0, "epilogue": 0, **kw}
    return LinearT(*(f[n] for n, _ in LinearT._fields_))


@pytest.mark.parametrize("bad", [dict(w=None), dict(scales=None), dict(out=None), dict(M=0), dict(M=-1), dict(out_stride=63), dict(epilogue=2), dict(epilogue=-1)], ids=str)
@pytest.mark.parametrize("at", [0, 2])
def test_tensors(bad, at):
    ts = [tensor(), tensor(), tensor()]; ts[at] = tensor(**bad)
    t = (LinearT * 3)(*ts)
    assert refused(lib.ibcu_linear_w8a8, t, 3, P, P, 64, 2) and refused(lib.ibcu_linear_w8a8_fp32, t, 3, P, 64, 2)


@pytest.mark.parametrize("n,N,B", [(0, 64, 1), (5, 64, 1), (-1, 64, 1), (1, 0, 1), (1, -16, 1), (1, 131073, 1), (1, 64, 0), (1, 64, -1), (1, 64, (1 << 20) + 1)])
def test_sizes(n, N, B):
    t = (LinearT * 5)(*[tensor() for _ in range(5)])
    assert refused(lib.ibcu_linear_w8a8, t, n, P, P, N, B) and refused(lib.ibcu_linear_w8a8_fp32, t, n, P, N, B)


@pytest.mark.parametrize("N,B", [(0, 1), (-1, 1), (1, 0), (1, -5)])
def test_quantiser(N, B):
    assert refused(lib.ibcu_quantize_rows_int8, P, P, P, N, B)


def test_null_vectors():
    t = (LinearT * 1)(tensor())
    assert refused(lib.ibcu_linear_w8a8, t, 1, None, P, 64, 1) and refused(lib.ibcu_linear_w8a8, t, 1, P, None, 64, 1)
    assert refused(lib.ibcu_linear_w8a8, None, 1, P, P, 64, 1) and refused(lib.ibcu_linear_w8a8_fp32, None, 1, P, 64, 1) and refused(lib.ibcu_linear_w8a8_fp32, t, 1, None, 64, 1)
    for i in range(3):
        a = [P] * 3; a[i] = None
        assert refused(lib.ibcu_quantize_rows_int8, *a, 64, 1)
    assert lib.ibcu_linear_w8a8(None, t, 1, P, P, 64, 1) == -1 and lib.ibcu_quantize_rows_int8(None, P, P, P, 64, 1) == -1 and lib.ibcu_linear_w8a8_fp32(None, t, 1, P, 64, 1) == -1
