"""Grouped products with more rows than their 32-bit tables and tile coordinates can number: refused before anything runs."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows", [2 ** 31 - 256, 2 ** 31, 2 ** 31 + 70])
def test_too_many_rows(rows, dtype):
    from honeycrisp_b200 import CUDABackend, NotImplementedByBackend
    be = CUDABackend(0)
    size = np.dtype(dtype).itemsize
    x, other = be.allocate(rows * size), be.allocate(rows * size)
    offsets = be.collection(np.array([0, 5, rows]), np.int64)
    matrices = be.constant(1.0, 2, dtype)
    launches = be.launchCount()
    with pytest.raises(NotImplementedByBackend, match="rows"):
        be.groupedMatmulWeightGrad(2, offsets, x, other, rows, 1, 1, dtype, out=matrices)
    with pytest.raises(NotImplementedByBackend, match="rows"):
        be.groupedMatmul(2, offsets, x, matrices, False, rows, 1, 1, dtype, out=other)
    assert be.launchCount() == launches
    assert (matrices.onCPU(dtype)[:2] == 1).all()
    be.checkDeviceStatus()
    be.close()


def test_too_long_a_contraction_for_tile_coordinates():
    """One row of float16 and a matrix that lies as TMA needs it: the tensor cores' product, whose contracted index is a 32-bit coordinate."""
    from honeycrisp_b200 import CUDABackend, NotImplementedByBackend
    be = CUDABackend(0)
    for inner in (2 ** 31, 2 ** 31 + 8):
        x, matrix = be.allocate(inner * 2), be.allocate(inner * 2)
        offsets, out = be.collection(np.array([0, 1]), np.int64), be.constant(1.0, 1, np.float16)
        launches = be.launchCount()
        with pytest.raises(NotImplementedByBackend, match="too large"):
            be.groupedMatmul(1, offsets, x, matrix, True, 1, inner, 1, np.float16, out=out)
        assert be.launchCount() == launches and out.onCPU(np.float16)[0] == 1
    be.checkDeviceStatus()
    be.close()
