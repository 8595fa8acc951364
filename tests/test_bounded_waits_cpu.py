"""The limits of the kernels' bounded waits: every library that is said to have one exports its controls."""
import re

import pytest

from rllm_b200.csrc import build, ops


def controls(source):
    return re.findall(r"^TC_DEFINE_WAIT_CONTROLS\((\w+)\)", (build.CSRC / source).read_text(), re.M)


@pytest.mark.parametrize("library", sorted(ops._WAIT_LIBRARIES))
def test_a_library_defines_its_controls(library):
    """... in the file whose kernels wait: the limit belongs to a translation unit."""
    sources = build.LIBRARIES[library][0]
    assert [ops._WAIT_LIBRARIES[library]] == [c for s in sources for c in controls(s)]


def test_every_waiting_kernel_is_listed():
    listed = {s for lib in ops._WAIT_LIBRARIES for s in build.LIBRARIES[lib][0]}
    for path in sorted(build.CSRC.glob("*.cu")):
        if re.search(r"\b(mbar_wait|warp_wait)\(", path.read_text()):
            assert path.name in listed and controls(path.name), path.name
