"""CPU checks of rules that the sources keep."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "scope_b200", "csrc")


def code_of(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def launched_as_dependents():
    return sorted(f for f in os.listdir(CSRC) if re.search(r"launch_dependent\s*\(", code_of(f)) and f != "ws_internal.h")


def test_the_rule_sees_the_paged_kernels():
    assert {"paged_decode.cuh", "paged_slots.cu", "rope_append.cu"} <= set(launched_as_dependents())


@pytest.mark.parametrize("name", launched_as_dependents())
def test_kernels_that_start_early_read_with_plain_loads(name):
    """A grid launched as a programmatic dependent starts while earlier ones still write; the read-only path is for memory
    that nobody writes while the kernel runs."""
    code = code_of(name)
    assert not re.findall(r"__ldg\s*\(|ld\.global\.nc|const\s+\w+\s*\*\s*(?:const\s+)?__restrict__", code)
