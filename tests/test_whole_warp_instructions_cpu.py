"""Instructions that a whole warp has to execute together, in the kernels' sources.

A warp that reaches an .aligned instruction with its lanes apart is undefined behaviour without a time limit, so no run shows it; the
rules that keep it from happening are checked where they are written down.
"""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "symplex_b200", "csrc")
FILES = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")))


def _code(path):
    with open(path) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def _device_functions(code):
    """(name, body) of the __device__ helpers."""
    for m in re.finditer(r"__device__ __forceinline__ [\w:]+ (\w+)\(", code):
        at = code.index("{", m.end())
        depth, end = 0, at
        while True:
            depth += {"{": 1, "}": -1}.get(code[end], 0) if not _in_string(code, at, end) else 0
            end += 1
            if depth == 0:
                break
        yield m.group(1), code[at:end]


def _in_string(code, start, pos):
    return code.count('"', start, pos) % 2 == 1


# mma.sync: between two __syncwarp of a step whose branches are uniform; tcgen05.wait::ld: directly behind the loads;
# relinquish: directly behind the allocation
EXEMPT = {"mma_bf16", "mma_bf16_zero", "tmem_ld_wait", "tmem_relinquish"}


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_lanes_are_brought_together_in_front(path):
    code = _code(path)
    found = 0
    for name, body in _device_functions(code):
        if ".aligned" not in body:
            continue
        found += len(re.findall(r"\.aligned", body))
        if name not in EXEMPT:
            assert "__syncwarp();" in body[:body.index(".aligned")], name
    assert found == len(re.findall(r"\.aligned", code)), "an .aligned instruction outside the helpers"


# barriers that every lane of a warp waits for: accumulators of the tensor core, tiles that a warp converts or evaluates
WHOLE_WARP = r"acc_full|main_full|corr_full|raw_full|op_empty|part_empty|part_full"


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_a_warp_leaves_a_wait_with_one_answer(path):
    code = _code(path)
    assert not re.findall(r"mbar_wait(?:<true>)?\(&(?:" + WHOLE_WARP + r")\b", code)
    if "tmem_ld_32x32(" in code and not path.endswith(".cuh"):
        assert "mbar_wait_warp(" in code or "mbar_wait_warp<true>(" in code
