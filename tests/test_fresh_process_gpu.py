"""Calls in a process that has made no others: what an earlier, larger call has arranged for a kernel (its opt-in to shared memory) is not there."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("what", ["decode", "decode_at", "few_tokens"])
def test_shared_memory_that_static_arrays_take_beyond_the_unasked_limit(what):
    """Heads of 96 in groups of 8, three positions of heads of 128 (the 4-bit cache), 12288 columns of four tokens and the like (INT8 x INT8): just below 48 KB of dynamic
    shared memory, beyond it with the kernel's own arrays."""
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tests", "_fresh_worker.py"), what], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fresh ok" in r.stdout, r.stderr[-2000:]
