"""Child process of the GPU tests: calls in a process that has made no others, where no larger call has opted a kernel in to its shared memory.

argv: <what>"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main():
    from libinferbit_b200 import Backend
    from tests import test_kv4_gpu, test_w8a8_gpu
    be = Backend(0)
    # Dynamic shared memory just below 48 KB, which the kernels' static arrays take beyond it
    steps = [(16, 2, 96, 40, 40, 1, 10000.0), (8, 8, 128, 50, 50, 3, 10000.0)]
    if sys.argv[1] == "decode":
        for shape in steps + [(5, 1, 96, 7, 7, 1, 10000.0)]:
            test_kv4_gpu.test_decode_step(be, *shape)
    elif sys.argv[1] == "decode_at":
        for n_heads, n_kv, hd, _, _, B, _ in steps:
            test_kv4_gpu.test_captured_at_a_device_place(be, n_heads, n_kv, hd, B, 256)
    else:
        for N, B in ((12288, 4), (16384, 3), (24576, 2), (49152, 1)):
            test_w8a8_gpu.run_both(be, np.random.default_rng(N), (1000, 24), N, B, False, 0)
    be.close()
    print("fresh ok")


main()
