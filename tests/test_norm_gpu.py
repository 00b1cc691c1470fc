"""Layer normalisation, forward and backward, against its formulas in float64."""
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


SHAPES = [(1, 1), (3, 1), (1, 2), (5, 7), (2, 8), (33, 31), (9, 64), (1, 256), (17, 257), (130, 512), (3, 1000), (7, 1024), (4, 2048),
          (5, 4096), (3, 4099), (2, 8192), (600, 96), (3, 8200), (2, 16384), (1, 20000), (2, 32768), (1, 40008), (1200, 136)]


def data(rows, cols, dtype, seed=0, offset=0.5):
    rng = np.random.default_rng(seed + rows * 31 + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(0.5 * rng.standard_normal(cols)) + offset).astype(dtype)
    w = (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    b = (0.2 * rng.standard_normal(cols)).astype(np.float32)
    g = rng.standard_normal((rows, cols)).astype(dtype)
    return x, w, b, g


def forward64(x, w, b, eps):
    x = x.astype(np.float64)
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / np.sqrt((d * d).mean(1) + eps)
    h = d * rstd[:, None]
    y = h * (1 if w is None else w.astype(np.float64)) + (0 if b is None else b.astype(np.float64))
    return y, mean, rstd, h


def sum_error(cols):
    """Relative to the sum of magnitudes, of a float32 sum of `cols` terms by threads of at most a few hundred terms each."""
    return (cols ** 0.5 + 64) * 2.0 ** -24


def forward_errors(x, h, rstd):
    """(mean's, rstd's relative, h's) float32 errors: the mean's carries to every difference; the variance is a sum of squares."""
    x = np.abs(x.astype(np.float64))
    n = x.shape[1]
    emean = x.mean(1) * sum_error(n) + 2.0 ** -149
    erstd = (sum_error(n) + 4 * 2.0 ** -24) + (emean * rstd) ** 2
    eh = (emean * rstd)[:, None] + np.abs(h) * erstd[:, None] + (x * rstd[:, None]) * 2.0 ** -23
    return emean, erstd, eh


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_forward(be, rows, cols, dtype):
    x, w, b, _ = data(rows, cols, dtype)
    mean, rstd = be.constant(0, rows, np.float32), be.constant(0, rows, np.float32)
    for ww, bb, pd in ((w, b, np.float32), (None, None, np.float32), (w.astype(np.float16), None, np.float16), (None, b, np.float32)):
        got = be.layerNorm(x, ww, bb, rows, cols, dtype, epsilon=1e-5, paramDType=pd, mean=mean, rstd=rstd)
        y, m, r, h = forward64(x, ww, bb, 1e-5)
        em, er, eh = forward_errors(x, h, r)
        ref.within(mean.onCPU(np.float32)[:rows], m, em, np.float32)
        ref.within(rstd.onCPU(np.float32)[:rows], r, r * er, np.float32)
        scale = 1 if ww is None else np.abs(ww.astype(np.float64))
        ref.within(got.onCPU(dtype)[: rows * cols], y, eh * scale + (np.abs(h) * scale + np.abs(y)) * 2.0 ** -23, dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward(be, rows, cols, dtype):
    x, w, b, g = data(rows, cols, dtype)
    _, m, r, _ = forward64(x, w, b, 1e-5)
    m32, r32 = m.astype(np.float32), r.astype(np.float32)
    h = (x.astype(np.float64) - m32[:, None].astype(np.float64)) * r32[:, None].astype(np.float64)   # of the stored statistics
    eh = (np.abs(x.astype(np.float64)) + np.abs(m)[:, None]) * r[:, None] * 2.0 ** -23
    g64, r64 = g.astype(np.float64), r32.astype(np.float64)
    for ww, pd in ((w, np.float32), (None, np.float32), (w.astype(np.float16), np.float16)):
        dx, dw, db = be.layerNormGrad(g, x, ww, m32, r32, rows, cols, dtype, paramDType=pd)
        wv = np.ones(cols) if ww is None else ww.astype(np.float64)
        gw = g64 * wv
        m0, m1 = gw.mean(1)[:, None], (gw * h).mean(1)[:, None]
        se = sum_error(cols)
        e0 = np.abs(gw).mean(1)[:, None] * (se + 2.0 ** -23)
        e1 = np.abs(gw * h).mean(1)[:, None] * (se + 2.0 ** -22) + (np.abs(gw) * eh).mean(1)[:, None]
        want = r64[:, None] * (gw - m0 - h * m1)
        err = r64[:, None] * (e0 + np.abs(h) * e1 + eh * np.abs(m1) + (np.abs(gw) + np.abs(m0) + np.abs(h * m1)) * 2.0 ** -22)
        ref.within(dx.onCPU(dtype)[: rows * cols], want, err, dtype)
        rs = rows * 2.0 ** -24 + 2.0 ** -22
        ref.within(dw.onCPU(pd)[:cols], (g64 * h).sum(0), np.abs(g64 * h).sum(0) * rs + (np.abs(g64) * eh).sum(0), pd)
        ref.within(db.onCPU(pd)[:cols], g64.sum(0), np.abs(g64).sum(0) * rs, pd)


def test_each_result_alone_and_none(be):
    rows, cols = 40, 264
    x, w, b, g = data(rows, cols, np.float16)
    _, m, r, _ = forward64(x, w, b, 1e-5)
    m, r = m.astype(np.float32), r.astype(np.float32)
    full = [t.onCPU(dt) for t, dt in zip(be.layerNormGrad(g, x, w, m, r, rows, cols, np.float16), (np.float16, np.float32, np.float32))]
    for want in range(3):
        asked = [want == 0, want == 1, want == 2]
        got = be.layerNormGrad(g, x, w, m, r, rows, cols, np.float16, out=None if asked[0] else False, weightGrad=asked[1], biasGrad=asked[2])
        assert [t is not None for t in got] == asked
        assert np.array_equal(got[want].onCPU(full[want].dtype), full[want])
    assert be.layerNormGrad(g, x, w, m, r, rows, cols, np.float16, out=False, weightGrad=False, biasGrad=False) == (None, None, None)


def test_no_rows(be):
    z = np.zeros((0, 16), np.float16)
    assert be.layerNorm(z, None, None, 0, 16, np.float16).byteCount == 0
    e = np.zeros(0, np.float32)
    _, dw, db = be.layerNormGrad(z, z, None, e, e, 0, 16, np.float16)
    assert not dw.onCPU(np.float32)[:16].any() and not db.onCPU(np.float32)[:16].any()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_constant_rows_large_offsets_and_non_finite(be, dtype):
    """A row of one value has variance zero; a large mean does not cancel the variance; NaN stays in its row."""
    rows, cols = 6, 520
    x, w, b, _ = data(rows, cols, dtype)
    x[0] = 3.0
    x[1] = (1000 + np.arange(cols) % 2).astype(dtype)
    x[2, 5] = np.nan
    x[3, 7] = np.inf
    got = be.layerNorm(x, w, b, rows, cols, dtype, epsilon=1e-5).onCPU(dtype).reshape(rows, cols)
    y, m, r, h = forward64(x[[0, 1, 4, 5]], w, b, 1e-5)
    _, er, eh = forward_errors(x[[0, 1, 4, 5]], h, r)
    ref.within(got[[0, 1, 4, 5]], y, eh * np.abs(w) + (np.abs(h * w) + np.abs(y)) * 2.0 ** -23, dtype)
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all()


def test_in_place_and_refusals(be):
    import torch
    rows, cols = 37, 512
    x, w, b, g = data(rows, cols, np.float16)
    want = be.layerNorm(x, w, b, rows, cols, np.float16).onCPU(np.float16)
    t = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    be.layerNorm(t, w, b, rows, cols, np.float16, out=t)
    be.sync()
    assert np.array_equal(t.cpu().numpy().reshape(-1), want[: rows * cols])
    m = torch.zeros(rows, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        be.layerNorm(t[1:], w, b, rows - 1, cols, np.float16, out=t)
    with pytest.raises(ValueError, match="overlaps"):
        be.layerNorm(t, w, b, rows, cols, np.float16, mean=m, rstd=m)
    with pytest.raises(ValueError, match="column"):
        be.layerNorm(t, None, None, rows, 0, np.float16)
    with pytest.raises(ValueError, match="epsilon"):
        be.layerNorm(t, w, b, rows, cols, np.float16, epsilon=-1.0)
    with pytest.raises(ValueError, match="smaller"):
        be.layerNorm(t, w[:-1], b, rows, cols, np.float16)
    with pytest.raises(ValueError, match="overlap"):
        be.layerNormGrad(t, x, w, m, m, rows, cols, np.float16, out=t)
    with pytest.raises(ValueError, match="contiguous"):
        be.layerNorm(t[:, :256], None, None, rows, 256, np.float16)


def test_gradient_against_differences(be):
    rng = np.random.default_rng(3)
    rows, cols = 5, 48
    x, w, b, g = data(rows, cols, np.float32)
    _, m, r, _ = forward64(x, w, b, 1e-5)
    dx, dw, db = be.layerNormGrad(g, x, w, m.astype(np.float32), r.astype(np.float32), rows, cols, np.float32)
    v, vw, vb = rng.standard_normal((rows, cols)), rng.standard_normal(cols), rng.standard_normal(cols)
    h = 1e-5
    f = lambda s: (forward64(x.astype(np.float64) + s * v, w + s * vw, b + s * vb, 1e-5)[0] * g).sum()  # noqa: E731
    diff = (f(h) - f(-h)) / (2 * h)
    along = (dx.onCPU(np.float32).reshape(rows, cols) * v).sum() + (dw.onCPU(np.float32) * vw).sum() + (db.onCPU(np.float32) * vb).sum()
    # float32 gradients: 2^-20 of the sum of magnitudes covers their errors; 1e-6 the quotient's
    room = (np.abs(dx.onCPU(np.float32).reshape(rows, cols) * v).sum() + np.abs(dw.onCPU(np.float32) * vw).sum() + np.abs(db.onCPU(np.float32) * vb).sum()) * 2.0 ** -18 + 1e-5
    assert abs(along - diff) <= room


def test_repeats_are_bitwise_equal(be):
    rows, cols = 1000, 1032
    x, w, b, g = data(rows, cols, np.float16)
    _, m, r, _ = forward64(x, w, b, 1e-5)
    m, r = m.astype(np.float32), r.astype(np.float32)
    a = [t.onCPU() for t in be.layerNormGrad(g, x, w, m, r, rows, cols, np.float16)]
    for _ in range(3):
        c = [t.onCPU() for t in be.layerNormGrad(g, x, w, m, r, rows, cols, np.float16)]
        assert all(np.array_equal(p, q) for p, q in zip(a, c))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols", [(3, 256), (400, 1024), (5, 4096), (330, 2048), (2, 8192)])
def test_rows_off_16_byte_boundaries(be, rows, cols, dtype):
    """The same rows one element further on: element accesses, the forward pass's sums in another order."""
    import torch
    x, w, b, g = data(rows, cols, dtype)
    tt = {np.float16: torch.float16, np.float32: torch.float32}[dtype]

    def off(v):
        t = torch.zeros(v.size + 1, dtype=tt, device="cuda")
        t[1:] = torch.from_numpy(v.reshape(-1)).cuda()
        return t[1:]

    xt, gt, out, dx = off(x), off(g), off(x), off(x)
    y, m, r, h = forward64(x, w, b, 1e-5)
    torch.cuda.synchronize()
    be.layerNorm(xt, w, b, rows, cols, dtype, out=out)
    _, dw, db = be.layerNormGrad(gt, xt, w, m.astype(np.float32), r.astype(np.float32), rows, cols, dtype, out=dx)
    be.sync()
    _, er, eh = forward_errors(x, h, r)
    ref.within(out.cpu().numpy(), y, eh * np.abs(w) + (np.abs(h * w) + np.abs(y)) * 2.0 ** -23, dtype)
    want = be.layerNormGrad(g, x, w, m.astype(np.float32), r.astype(np.float32), rows, cols, dtype)
    # two orders of the same float32 sums
    room = np.abs(g.astype(np.float64) * w).mean(1)[:, None] * (1 + np.abs(h)) * r[:, None] * 4 * sum_error(cols) + np.abs(g * w) * r[:, None] * 2.0 ** -21
    ref.within(dx.cpu().numpy(), want[0].onCPU(dtype)[: rows * cols].astype(np.float64), room + 2 * ref.HALF_STEP[dtype] * np.abs(want[0].onCPU(dtype)[: rows * cols].reshape(rows, cols).astype(np.float64)), dtype)
    sums = np.abs(g.astype(np.float64) * h).sum(0) * (rows * 2.0 ** -23 + 2.0 ** -21)
    ref.within(dw.onCPU(np.float32)[:cols], want[1].onCPU(np.float32)[:cols].astype(np.float64), sums + np.abs(g).astype(np.float64).sum(0) * 2.0 ** -22, np.float32)
    ref.within(db.onCPU(np.float32)[:cols], want[2].onCPU(np.float32)[:cols].astype(np.float64), np.abs(g).astype(np.float64).sum(0) * rows * 2.0 ** -23, np.float32)
