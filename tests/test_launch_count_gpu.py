"""The context counts the kernels that it launches, not those that it might have."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_activation_gradient():
    from honeycrisp_b200 import CUDABackend
    be = CUDABackend(0)
    for rows, cols, sums, launches in [(64, 96, True, 1), (3, 5, True, 1), (64, 96, False, 1), (65, 96, True, 2), (1000, 33, True, 2), (0, 8, True, 1), (0, 8, False, 0)]:
        x = be.constant(0.5, max(1, rows * cols), np.float32)
        before = be.launchCount()
        be.activationGrad(x, x, rows, cols, np.float32, "gelu", biasGrad=sums)
        assert be.launchCount() - before == launches, (rows, cols, sums)
    be.checkDeviceStatus()
    be.close()


def test_layer_norm_gradient_and_products_of_few_rows():
    from honeycrisp_b200 import CUDABackend
    be = CUDABackend(0)
    x, s = be.constant(0.5, 40 * 264, np.float32), be.constant(1.0, 264, np.float32)
    for sums, launches in [(True, 2), (False, 1)]:
        before = be.launchCount()
        be.layerNormGrad(x, x, s, s, s, 40, 264, np.float32, weightGrad=sums, biasGrad=sums)
        assert be.launchCount() - before == launches
    before = be.launchCount()
    be.matmulEpilogue(x, False, x, False, 4, 40, 264, np.float32)   # the product's parts, and their sum
    assert be.launchCount() - before == 2
    be.checkDeviceStatus()
    be.close()
