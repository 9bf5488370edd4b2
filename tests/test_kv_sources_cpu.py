"""CPU: the kernels over the quantised cache begin while the kernels before them may still run (griddepcontrol), so nothing
that those write is read by the path for memory that stays as it is during a kernel."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gemlite_b200", "csrc")


@pytest.mark.parametrize("name", sorted(f for f in os.listdir(CSRC) if f.startswith("gl_kv") and f.endswith((".cu", ".cuh"))))
def test_no_read_only_loads(name):
    code = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    assert not re.search(r"__ldg\s*\(|ld\.global\.nc|__restrict__", code)
