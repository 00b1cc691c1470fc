"""The C entry points of the feed-forward operators up to their launches, on the host: hc_ops.cu, which holds no device code, built by the host
compiler over stubs that count launches (tests/cpp/operators_on_stubs.cpp)."""
import ctypes
import os
import shutil
import subprocess

import pytest

from honeycrisp_b200 import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CTX, A, B, OUT, OFFSETS = 64, 1 << 40, 1 << 44, 1 << 48, 4096


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    if not os.path.exists(include) or shutil.which("g++") is None:
        pytest.skip("no host compiler or CUDA headers")
    path = str(tmp_path_factory.mktemp("stubs") / "operators.so")
    subprocess.check_call(["g++", "-std=c++17", "-w", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", include, "-o", path, "-x", "c++", os.path.join(ROOT, "tests", "cpp", "operators_on_stubs.cpp"),
                           "-x", "c++", os.path.join(ROOT, "honeycrisp_b200", "csrc", "hc_ops.cu")])
    lib = ctypes.CDLL(path)
    for name, (res, args) in L.SIGNATURES.items():
        if hasattr(lib, name):
            getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    lib.stub_message.restype = ctypes.c_char_p
    return lib


@pytest.mark.parametrize("dtype", [L.HC_F16, L.HC_F32])
def test_groups_of_more_rows_than_tile_coordinates_number(lib, dtype):
    """Row numbers are 32-bit on the device, and the last slab's copies start up to a tile behind them."""
    for rows, status in [(5, L.HC_OK), (2 ** 31 - 257, L.HC_OK), (2 ** 31 - 256, L.HC_ERR_NOT_IMPLEMENTED), (2 ** 31, L.HC_ERR_NOT_IMPLEMENTED),
                         (2 ** 31 + 70, L.HC_ERR_NOT_IMPLEMENTED), (2 ** 41, L.HC_ERR_NOT_IMPLEMENTED)]:
        assert lib.hc_grouped_matmul_weight_grad(CTX, dtype, 2, OFFSETS, A, B, rows, 1, 1, OUT) == status
        assert (lib.stub_enqueued() > 0) == (status == L.HC_OK)
        assert lib.hc_grouped_matmul(CTX, dtype, 2, OFFSETS, A, B, 0, rows, 1, 1, OUT) == status
        assert (lib.stub_enqueued() > 0) == (status == L.HC_OK)
