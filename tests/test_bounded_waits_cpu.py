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


def test_a_wait_that_ran_out_is_named(monkeypatch):
    """Every code that a kernel writes when it gives up a wait has its words; another one is still reported."""
    import torch
    words = {}
    for path in sorted(build.CSRC.glob("*.cu")):
        if path.name not in {s for lib in ops._WAIT_LIBRARIES for s in build.LIBRARIES[lib][0]}:
            continue
        for body in re.findall(r"^enum \{([^}]*_ERR_[^}]*)\}", path.read_text(), re.M):
            words.update({int(v): name for name, v in re.findall(r"(\w+_ERR_\w+) = (\d+)", body)})
    assert set(words) >= {1, 2, 3, 21, 31, 34}
    word = torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(ops, "error_word", lambda device: word)
    for code in sorted(words):
        word.fill_(code)
        with pytest.raises(ops.KernelError, match=rf"bounded wait ran out \(code {code}: [a-z]"):
            ops.check_device_errors()
        assert int(word) == 0
    word.fill_(99)
    with pytest.raises(ops.KernelError, match=r"bounded wait ran out \(code 99\)"):
        ops.check_device_errors()
