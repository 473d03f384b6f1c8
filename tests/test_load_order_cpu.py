"""Kernels that overlap the launch in front of them read what it wrote with ordered loads."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eider_b200", "csrc")
WAITS = re.compile(r"griddepcontrol\.wait|griddep_wait\(\)|griddep_begin\(\)")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def files():
    return sorted(f for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh")))


# the loaders that waiting kernels of other files use
SHARED = {"quant_block.cuh"}


@pytest.mark.parametrize("name", [f for f in files() if f in SHARED or WAITS.search(code(f))])
def test_no_read_only_load_of_what_the_launch_in_front_wrote(name):
    """To the compiler a read-only load (__ldg) has no order with griddepcontrol.wait.  Files with kernels that wait there do without; the
    decode step of a routed layer reads its weights so, which never change while kernels run, but neither x nor the router's logits."""
    loads = re.findall(r"__ldg\([^;]*", code(name))
    if name == "decode_moe.cu":
        loads = [load for load in loads if re.search(r"\ba\.(x|logits|act)\b", load)]
    assert not loads, loads
