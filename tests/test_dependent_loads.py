"""CPU suite: kernels that are resident before the launch in front has ended read their inputs with plain loads.

Read-only loads promise that the data do not change while the kernel runs, which an output of the launch in front does.
Weights and their scales, laid out once, are the only data of the 8-bit products that may be read so."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "fastertnn_b200" / "csrc"


def code(name):
    """The source without its comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", (CSRC / name).read_text(), flags=re.S)


@pytest.mark.parametrize("name", ["route.cu", "rows_i8.cu", "gemm_i8.cu"])
def test_read_only_loads_take_constants(name):
    source = code(name)
    assert "griddepcontrol.wait" in source
    assert all(what.startswith("p.w_scale") for what in re.findall(r"__ldg\(([^)]*)", source))
    # the one read-only load that is written out is that of the weights' tiles
    users = re.findall(r"\bload_32b\(([^,]*)", source)
    assert ("ld.global.nc" in source) == bool(users)
    assert all(u.startswith(("const int8_t*", "tile")) for u in users)


@pytest.mark.parametrize("name", ["route.cu", "rows_i8.cu", "gemm_i8.cu"])
def test_inputs_are_not_declared_unaliased(name):
    kernels = code(name).split("__global__")[1:]
    assert kernels
    for kernel in kernels:
        head, body = kernel.split("{", 1)
        if "griddepcontrol.wait" in body:
            assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", head), head
