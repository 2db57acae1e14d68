"""INT8 weights that a kernel has just written, read from the source (no GPU).

Products ask for their weights ahead of the wait for the launch before them. What writes a tensor's weights must therefore start nobody early: a launch that
executes no griddepcontrol.launch_dependents is complete before its successor begins."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "libinferbit_b200", "csrc")
CODE = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "w8a8.cu")).read())


def test_a_callers_codes_are_written_before_anyone_starts():
    kernel = CODE[CODE.index("quantize_rows_kernel("):].split("\n}\n")[0]
    starts = re.findall(r"[^\n]*pdl_launch_dependents\(\)", kernel)
    assert [s.strip() for s in starts] == ["if (OWN) pdl_launch_dependents()"]
    public = CODE[CODE.index('int ibcu_quantize_rows_int8('):].split("\n}\n")[0]
    assert "quantize<false>(" in public and "quantize<true>" not in public
    launch = CODE[CODE.index("int quantize("):].split("\n}\n")[0]
    assert re.findall(r"quantize_rows_kernel<\w+, (\w+)>", launch) == ["OWN", "OWN"]


def test_products_read_weights_early():
    """The reason: if this no longer holds, the rule above may go."""
    few = CODE[CODE.index("w8a8_few_kernel("):].split("\n}\n")[0]
    assert few.index("fetch(0)") < few.index("pdl_wait()")
