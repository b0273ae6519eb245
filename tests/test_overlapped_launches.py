"""Kernels that may begin while the kernel before still runs read global memory by loads that stay behind their wait (CPU only).

A read-only load promises that nothing writes the memory as long as the kernel lives; with an overlapped launch the kernel before
may still be writing it, and the compiler may move such a load in front of the wait.  The order cannot be provoked from outside, so
this reads the sources."""
import glob
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "quadmul_b200", "csrc")
READ_ONLY = re.compile(r"__ldg\(|__ldcs\(|__ldca\(|ld\.global\.nc|const\s+[\w:]+\s*\*\s*__restrict__")


def code(path):
    """The file without its comments."""
    with open(path) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def overlapped():
    """(file, part, text): every kernel that waits for the kernel before, and the functions in front of a file's first kernel."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        parts = code(path).split("__global__")
        waits = [k for k, part in enumerate(parts) if "grid_dependency_wait" in part]
        for k in [0, *waits] if waits else []:
            yield os.path.basename(path), k, parts[k]


CASES = list(overlapped())


def test_there_are_such_kernels():
    assert {"qm_gemv.cu", "qm_gemm_rmma.cu", "qm_gemm_dec.cu", "qm_gemm_tc2.cu", "qm_w4_rows.cu", "qm_w4_tc.cu", "qm_w4_pad.cu"} <= {c[0] for c in CASES}


@pytest.mark.parametrize("name,part,text", CASES, ids=[f"{c[0]}-{c[1]}" for c in CASES])
def test_loads_stay_behind_the_wait(name, part, text):
    assert not READ_ONLY.findall(text)


def test_shared_helpers_of_the_products():
    """The experts' segments are read by the products themselves."""
    text = code(os.path.join(CSRC, "qm_w4.cuh"))
    assert not READ_ONLY.findall(text) and "ptx::ld_behind_wait(offsets" in text


@pytest.mark.parametrize("name", ["qm_w4_rows.cu", "qm_w4_tc.cu", "qm_w4_pad.cu"])
def test_products_let_successors_begin_behind_their_own_wait(name):
    """So that no kernel is resident while the last but one before it still writes."""
    for part in code(os.path.join(CSRC, name)).split("__global__")[1:]:
        if "grid_dependency_wait" in part:
            assert 0 <= part.index("grid_dependency_wait") < part.index("grid_launch_dependents")
