"""Backward pass of the layer norm on rows whose mean is thousands of times their spread, against the formulas in float64 of the statistics that
were handed in: x - mean is then a small difference of large numbers, exact but for one rounding, and so is all that follows from it."""
import numpy as np
import pytest

import operator_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    from honeycrisp_b200 import CUDABackend
    b = CUDABackend(0)
    yield b
    b.checkDeviceStatus()
    b.close()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("cols", [200, 264, 999, 1024, 2048, 4096, 8192, 8200])
def test_large_means(be, cols, dtype):
    rows = 37
    rng = np.random.default_rng(cols)
    # means of 25 to 190 times the spread in float16, 200 to 60000 times in float32
    offset = np.exp(rng.uniform(np.log(200), np.log(1500 if dtype == np.float16 else 60000), rows))[:, None]
    x = (offset * np.where(np.arange(rows) % 2, 1, -1)[:, None] + rng.standard_normal((rows, cols)) * (8 if dtype == np.float16 else 1)).astype(dtype)
    x[5] = 1000.1            # one value: x - mean is zero, and rstd what epsilon leaves
    w = (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    g = rng.standard_normal((rows, cols)).astype(dtype)
    x64, g64 = x.astype(np.float64), g.astype(np.float64)
    mean = x64.mean(1).astype(np.float32)
    d = x64 - mean[:, None].astype(np.float64)
    rstd = (1 / np.sqrt((d * d).mean(1) + 1e-5)).astype(np.float32)
    r = rstd[:, None].astype(np.float64)
    h = d * r
    dx, dw, db = be.layerNormGrad(g, x, w, mean, rstd, rows, cols, dtype)
    # h: the difference's rounding and the product's, 2^-24 of the value each
    eh = np.abs(h) * 2.0 ** -23 * (1 + 2.0 ** -20)
    # a float32 sum of `cols` terms by threads of a few hundred each, then in a tree
    sums = (cols ** 0.5 + 64) * 2.0 ** -24
    gw = g64 * w.astype(np.float64)
    m0, m1 = gw.mean(1)[:, None], (gw * h).mean(1)[:, None]
    e0 = np.abs(gw).mean(1)[:, None] * (sums + 2.0 ** -23)
    e1 = np.abs(gw * h).mean(1)[:, None] * (sums + 2.0 ** -22) + (np.abs(gw) * eh).mean(1)[:, None]
    want = r * (gw - m0 - h * m1)
    err = r * (e0 + np.abs(h) * e1 + eh * np.abs(m1) + (np.abs(gw) + np.abs(m0) + np.abs(h * m1)) * 2.0 ** -22)
    ref.within(dx.onCPU(dtype)[: rows * cols], want, err, dtype)
    along = rows * 2.0 ** -24 + 2.0 ** -22
    ref.within(dw.onCPU(np.float32)[:cols], (g64 * h).sum(0), np.abs(g64 * h).sum(0) * along + (np.abs(g64) * eh).sum(0), np.float32)
    ref.within(db.onCPU(np.float32)[:cols], g64.sum(0), np.abs(g64).sum(0) * along, np.float32)
