"""Kernels that may start before the kernel in front has ended must not read through the non-coherent cache: such loads require memory that
does not change while the kernel runs, and what they read may be what that other kernel still writes."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "honeycrisp_b200", "csrc")


def code(path):
    with open(path) as f:
        text = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def early_starting():
    """Sources of kernels launched by programmatic dependent launch: those that wait for the kernel in front themselves."""
    return [p for p in glob.glob(os.path.join(CSRC, "*.cu*")) if "pdl_wait()" in code(p)]


def test_no_loads_through_the_non_coherent_cache():
    sources = early_starting()
    assert {"gemm_skinny.cu", "gemm_tc.cu", "tc_kernel.cuh", "norm.cu", "activation.cu", "adamw.cu"} <= {os.path.basename(p) for p in sources}
    for path in sources + [os.path.join(CSRC, "epilogue.cuh")]:   # device functions of several of them
        found = re.findall(r"__ldg\w*|ld\.global\.nc|__restrict__", code(path))
        assert not found, f"{os.path.basename(path)}: {found}"
