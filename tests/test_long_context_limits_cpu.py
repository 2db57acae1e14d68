"""Sizes at the end of what an int holds, which the 4-bit cache and INT8 x INT8 calls refuse before anything is launched (see test_kv4_cpu.py for the zeroed context)."""
import pytest

from libinferbit_b200 import LinearT
from tests.test_w8a8_cpu import P, lib, refused, tensor

pytestmark = pytest.mark.skipif(lib.ibcu_device_count() > 0, reason="with a GPU, a call that is not refused would launch")


@pytest.mark.parametrize("N", [(1 << 30) + 1, 2**31 - 512, 2**31 - 1])
def test_rows_whose_index_would_wrap(N):
    assert refused(lib.ibcu_quantize_rows_int8, P, P, P, N, 1)


@pytest.mark.parametrize("M", [2**31 - 255, 2**31 - 128, 2**31 - 1])
def test_tensors_whose_tiles_would_wrap(M):
    for ts in ([tensor(M=M, out_stride=2**31 - 1)], [tensor(), tensor(M=M, out_stride=2**31 - 1)]):
        t = (LinearT * len(ts))(*ts)
        assert refused(lib.ibcu_linear_w8a8, t, len(ts), P, P, 16, 1) and refused(lib.ibcu_linear_w8a8_fp32, t, len(ts), P, 16, 1)
