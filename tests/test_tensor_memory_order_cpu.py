"""Tensor memory is taken before the next kernel is let in, read off the sources (no GPU).

``tcgen05.alloc`` waits until the columns are free.  A kernel that let its successor start first
(``griddepcontrol.launch_dependents``) and allocated afterwards could find the columns held by that
successor, which in turn waits for it to end; neither wait has a limit.
"""

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "iron_b200" / "csrc"


def allocating_kernels():
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        starts = [m.start() for m in re.finditer(r"__global__", text)] + [len(text)]
        for a, b in zip(starts, starts[1:]):
            if "tcgen05.alloc" in text[a:b]:
                yield pytest.param(text[a:b], id=f"{path.stem}-{text[:a].count('__global__')}")


@pytest.mark.parametrize("kernel", list(allocating_kernels()))
def test_columns_are_taken_before_dependents_are_launched(kernel):
    launch = kernel.find("pdl_launch()")
    assert launch < 0 or kernel.find("tcgen05.alloc") < launch
