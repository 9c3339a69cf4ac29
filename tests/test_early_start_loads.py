"""CPU check of the kernels that start while the kernel before them on the stream still
runs (programmatic stream serialization): nothing there is read by read-only
loads (__ldg, ld.global.nc, const __restrict__ pointers), which promise that nobody
writes the data while the kernel is resident."""
import os
import re

import autoresearch2_b200

CSRC = os.path.join(os.path.dirname(autoresearch2_b200.__file__), "csrc")


def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_kernels_that_start_early_use_no_read_only_loads():
    waiting = [f for f in sorted(os.listdir(CSRC)) if f.endswith(".cu") and "grid_dependency_wait()" in source(f)]
    assert waiting == ["fewrows.cu", "narrow.cu"]
    for name in waiting:
        assert not re.findall(r"__ldg|ld\.global\.nc|__restrict__", source(name)), name
