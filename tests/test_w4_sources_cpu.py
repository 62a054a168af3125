"""Rules that the sources of the 4-bit weight kernels keep and that no run can show to be broken."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hipgemm_b200", "csrc")
KERNELS = ["w4.cu", "w4.cuh", "w4_tc.cu", "w4_tc.cuh", "moe.cu"]


def _code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", KERNELS)
def test_no_non_coherent_loads(name):
    """These kernels are launched with programmatic stream serialization: the kernel before them may be writing their
    operands when they start, so that no load may take the path for data that never changes while a kernel runs."""
    assert re.findall(r"__ldg|ld\.global[.\w:]*\.nc|\btex1D|__restrict__|__restrict\b", _code(name)) == []


def test_what_is_read_before_the_wait_comes_from_l2():
    """The experts' second and third kernel read ids and weights before griddepcontrol.wait.  What wrote them has ended
    (the first kernel waits before it triggers), but only L2 is sure to show it to a kernel that has not waited."""
    code = _code("moe.cu")
    assert re.findall(r"p\.(?:ids|weights)\s*\[[^\]]*\](?!\s*=)", code) == []
    assert len(re.findall(r"__ldcg\((?:given|p\.ids|p\.weights) \+", code)) == 3
