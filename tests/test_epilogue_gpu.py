"""Products with bias, activation and residual in their epilogue, and the gradients through an activation."""
import numpy as np
import pytest

import operator_reference as ref

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


@pytest.fixture(scope="module")
def be():
    from honeycrisp_b200 import CUDABackend
    b = CUDABackend(0)
    yield b
    b.checkDeviceStatus()
    b.close()


@pytest.fixture(scope="module")
def diag():
    from honeycrisp_b200 import CUDABackend
    b = CUDABackend(0, diagnostics=True)
    yield b
    b.checkDeviceStatus()
    b.close()


def operands(rng, rows, inner, cols, dtype, ta=False, tb=False):
    a = rng.standard_normal((rows, inner)).astype(dtype)
    b = (rng.standard_normal((inner, cols)) / np.sqrt(max(1, inner))).astype(dtype)
    return a, b, (np.ascontiguousarray(a.T) if ta else a), (np.ascontiguousarray(b.T) if tb else b)


def forward_case(be, rows, inner, cols, dtype, act, bias, residual, pre, ta=False, tb=False, seed=0):
    rng = np.random.default_rng(seed + rows * 7 + inner * 3 + cols)
    a, b, sa, sb = operands(rng, rows, inner, cols, dtype, ta, tb)
    bv = rng.standard_normal(cols).astype(dtype) if bias else None
    rv = rng.standard_normal((rows, cols)).astype(dtype) if residual else None
    pv = be.constant(7.0, rows * cols, dtype) if pre else None
    out = be.matmulEpilogue(sa, ta, sb, tb, rows, inner, cols, dtype, activation=act, bias=bv, residual=rv, pre=pv)
    z = a.astype(np.float64) @ b.astype(np.float64)
    err = ref.product_error(a, b, dtype)
    if bias:
        z = z + bv.astype(np.float64)
        err = err + np.abs(z) * 2.0 ** -24
    y = ref.activation(z, act)
    yerr = err * 1.13 + np.abs(y) * (ref.ACT_RELATIVE[dtype] if act in ("gelu", "gelu_tanh", "silu") else 0)   # slopes stay below 1.13
    if residual:
        y = y + rv.astype(np.float64)
        yerr = yerr + np.abs(y) * 2.0 ** -24
    ref.within(out.onCPU(dtype)[: rows * cols], y, yerr, dtype)
    if pre:
        ref.within(pv.onCPU(dtype)[: rows * cols], z, err, dtype)
    return out


SHAPES = [(1, 1, 1), (1, 64, 257), (3, 40, 65), (4, 4096, 512), (5, 520, 4099), (64, 128, 96), (129, 72, 130), (257, 320, 264),
          (300, 1024, 1032), (128, 4096, 128), (40, 8192, 40), (1000, 96, 1001), (520, 2048, 1536)]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,inner,cols", SHAPES)
def test_every_activation_with_everything(be, rows, inner, cols, dtype):
    for i, act in enumerate(ACTS):
        forward_case(be, rows, inner, cols, dtype, act, True, True, True, ta=bool(i & 1), tb=bool(i & 2))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("bias,residual,pre", [(False, False, False), (True, False, False), (False, True, False), (False, False, True)])
def test_each_extra_alone(be, bias, residual, pre, dtype):
    for shape in [(3, 5, 7), (130, 200, 264), (256, 1024, 96)]:
        forward_case(be, *shape, dtype, "gelu", bias, residual, pre)


@pytest.mark.parametrize("shape", range(1, 7))
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_every_tile_shape(diag, monkeypatch, shape, dtype):
    monkeypatch.setenv("HC_TC_SHAPE", str(shape))
    monkeypatch.setenv("HC_TC_SPLITS", "1")
    monkeypatch.setenv("HC_TC_WIDE_MIN_KB", "1")
    for rows, inner, cols in [(300, 200, 1100), (520, 1024, 1032), (257, 640, 1025)]:
        forward_case(diag, rows, inner, cols, dtype, "gelu_tanh", True, True, True)


@pytest.mark.parametrize("inner", [2048, 4100])
def test_long_contractions_on_the_widest_tile(diag, monkeypatch, inner):
    """256x256 tiles whose pipeline and epilogue change with the contraction's length, several tiles a CTA pair."""
    monkeypatch.setenv("HC_TC_SHAPE", "2")
    monkeypatch.setenv("HC_TC_SPLITS", "1")
    for extras in [(True, False, False), (True, True, False), (True, False, True), (True, True, True)]:
        forward_case(diag, 300, inner, 600, np.float16, "gelu", *extras)
    rng = np.random.default_rng(inner)
    a, b, _, _ = operands(rng, 300, inner, 600, np.float16)
    pre = rng.standard_normal((300, 600)).astype(np.float16)
    out = diag.matmulEpilogue(a, False, b, False, 300, inner, 600, np.float16, activation="silu", gradPre=pre)
    d = ref.slope(pre.astype(np.float64), "silu")
    z = a.astype(np.float64) @ b.astype(np.float64)
    ref.within(out.onCPU(np.float16)[: 300 * 600], z * d, ref.product_error(a, b, np.float16) * np.abs(d) + np.abs(z) * 4e-5, np.float16)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_cut_contractions(diag, monkeypatch, dtype):
    for parts in (2, 5):
        monkeypatch.setenv("HC_TC_SPLITS", str(parts))
        for rows, inner, cols in [(130, 1024, 136), (257, 1000, 131)]:
            forward_case(diag, rows, inner, cols, dtype, "gelu", True, True, True)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("tb", [False, True])
def test_few_columns_and_long_contractions(be, dtype, tb):
    """A result of one to three columns over a long contraction: one tile, cut into parts."""
    for rows, inner, cols in [(9, 17, 1), (48, 121, 20), (20, 16, 7), (9, 256, 1), (16, 300, 3), (40, 2048, 2), (8, 1500, 1), (1, 40000, 5), (7, 1030, 640)]:
        forward_case(be, rows, inner, cols, dtype, "silu", True, True, False, tb=tb)


def test_same_buffers_with_other_extras(be):
    """Repeats with the same operands and result but another bias, residual, kept tensor or activation: nothing of an earlier call stays."""
    import torch
    rng = np.random.default_rng(6)
    rows, inner, cols = 256, 256, 512
    a, b, _, _ = operands(rng, rows, inner, cols, np.float16)
    ad, bd = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()
    extras = [torch.from_numpy(rng.standard_normal(cols).astype(np.float16)).cuda() for _ in range(2)]
    wide = [torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float16)).cuda() for _ in range(2)]
    kept = [torch.zeros(rows, cols, dtype=torch.float16, device="cuda") for _ in range(2)]
    out = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    z = a.astype(np.float64) @ b.astype(np.float64)
    err = ref.product_error(a, b, np.float16) + 2.0 ** -20
    torch.cuda.synchronize()
    for act in ("none", "relu"):
        for bias in (None, *extras):
            for res in (None, *wide):
                for pre in (None, *kept):
                    if pre is not None:
                        pre.zero_()
                        torch.cuda.synchronize()
                    be.matmulEpilogue(ad, False, bd, False, rows, inner, cols, np.float16, activation=act, bias=bias, residual=res, pre=pre, out=out)
                    be.sync()
                    want = z if bias is None else z + bias.cpu().numpy().astype(np.float64)
                    if pre is not None:
                        ref.within(pre.cpu().numpy(), want, err, np.float16)
                    want = ref.activation(want, act) + (0 if res is None else res.cpu().numpy().astype(np.float64))
                    ref.within(out.cpu().numpy(), want, err, np.float16)
    for grad in wide:
        for act in ("relu", "silu"):
            be.matmulEpilogue(ad, False, bd, False, rows, inner, cols, np.float16, activation=act, gradPre=grad, out=out)
            be.sync()
            d = ref.slope(grad.cpu().numpy().astype(np.float64), act)
            ref.within(out.cpu().numpy(), z * d, err * 1.2 + np.abs(z) * 4e-5, np.float16)


def test_two_contexts_at_once(be):
    """Two contexts on two streams, the same inputs, calls enqueued in turn: each has its own work area."""
    import torch
    from honeycrisp_b200 import CUDABackend
    rng = np.random.default_rng(1)
    rows, inner, cols = 4, 4096, 1000                     # partial sums in the work area
    a, b, _, _ = operands(rng, rows, inner, cols, np.float16)
    ad, bd = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()
    others = [CUDABackend(0) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in others]
    outs = [torch.empty(8, rows, cols, dtype=torch.float16, device="cuda") for _ in others]
    torch.cuda.synchronize()
    for o, s in zip(others, streams):
        o.useStream(s.cuda_stream)
    for i in range(8):
        for o, out in zip(others, outs):
            o.matmulEpilogue(ad, False, bd, False, rows, inner, cols, np.float16, activation="gelu" if i % 2 else "relu", out=out[i], mark=False)
    torch.cuda.synchronize()
    for i in range(8):
        want = be.matmulEpilogue(a, False, b, False, rows, inner, cols, np.float16, activation="gelu" if i % 2 else "relu").onCPU(np.float16)
        for out in outs:
            assert np.array_equal(out[i].cpu().numpy().reshape(-1), want[: rows * cols])
    for o in others:
        o.checkDeviceStatus()
        o.close()


def test_empty_sizes(be):
    """An empty contraction leaves bias, activation and residual; no rows or no columns leave nothing to do."""
    forward_case(be, 5, 0, 9, np.float16, "silu", True, True, True)
    assert be.matmulEpilogue(np.zeros((0, 4), np.float32), False, np.zeros((4, 3), np.float32), False, 0, 4, 3, np.float32).byteCount == 0
    be.matmulEpilogue(np.zeros((4, 4), np.float32), False, np.zeros((4, 0), np.float32), False, 4, 4, 0, np.float32)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,inner,cols", [(1, 1, 1), (7, 33, 130), (64, 64, 64), (300, 520, 1032), (130, 1000, 131), (256, 4096, 256)])
def test_gradient_form(be, rows, inner, cols, dtype):
    rng = np.random.default_rng(rows + cols)
    a, b, sa, sb = operands(rng, rows, inner, cols, dtype, False, True)
    pre = (rng.standard_normal((rows, cols)) * 2).astype(dtype)
    z = a.astype(np.float64) @ b.astype(np.float64)
    err = ref.product_error(a, b, dtype)
    for act in ACTS:
        out = be.matmulEpilogue(sa, False, sb, True, rows, inner, cols, dtype, activation=act, gradPre=pre)
        d = ref.slope(pre.astype(np.float64), act)
        # the slope adds two terms, each off by its own relative error
        derr = (np.abs(d) + np.abs(pre.astype(np.float64)) * 0.8) * ref.ACT_RELATIVE[dtype] if act in ("gelu", "gelu_tanh", "silu") else 0 * d
        ref.within(out.onCPU(dtype)[: rows * cols], z * d, err * np.abs(d) + np.abs(z) * derr + err * derr, dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 4096), (3, 7), (17, 64), (130, 257), (1000, 40), (4099, 8), (600, 1032)])
def test_activation_grad_and_bias_grad(be, rows, cols, dtype):
    rng = np.random.default_rng(rows * cols)
    g = rng.standard_normal((rows, cols)).astype(dtype)
    pre = (rng.standard_normal((rows, cols)) * 2).astype(dtype)
    for act in ACTS:
        out, db = be.activationGrad(g, pre, rows, cols, dtype, act)
        z, g64 = pre.astype(np.float64), g.astype(np.float64)
        d = ref.slope(z, act)
        derr = (np.abs(d) + np.abs(z) * 0.8) * ref.ACT_RELATIVE[dtype] if act in ("gelu", "gelu_tanh", "silu") else 0 * d
        err = np.abs(g64) * derr + np.abs(g64 * d) * 2.0 ** -22
        ref.within(out.onCPU(dtype)[: rows * cols], g64 * d, err, dtype)
        # summed in float32: rows 2^-24 of the sum of magnitudes at most
        ref.within(db.onCPU(np.float32)[:cols], (g64 * d).sum(0), err.sum(0) + rows * 2.0 ** -24 * np.abs(g64 * d).sum(0), np.float32)
    out, db = be.activationGrad(g, pre, rows, cols, dtype, "gelu", biasGrad=False)
    assert db is None


def test_activation_grad_without_rows(be):
    out, db = be.activationGrad(np.zeros((0, 9), np.float16), np.zeros((0, 9), np.float16), 0, 9, np.float16, "gelu")
    assert np.array_equal(db.onCPU(np.float32)[:9], np.zeros(9, np.float32))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_special_values(be, dtype):
    """NaN and infinities where the formulas put them, the tails where they vanish, and slopes that stay finite."""
    top = float(np.finfo(dtype).max)
    vals = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, top, -top, 1e-4, -1e-4, 20.0, -20.0, 100.0, -100.0, 5.0, -5.0, 1.0], dtype)
    rows, inner, cols = 64, 64, vals.size * 4
    a = np.zeros((rows, inner), dtype)
    b = np.zeros((inner, cols), dtype)
    bias = np.tile(vals, 4)
    z = bias.astype(np.float64)
    for act in ACTS:
        got = be.matmulEpilogue(a, False, b, False, rows, inner, cols, dtype, activation=act, bias=bias).onCPU(dtype).reshape(rows, cols)
        with np.errstate(all="ignore"):
            want = ref.activation(z, act)
        finite = np.isfinite(want)
        assert np.array_equal(np.isnan(got[0]), np.isnan(want)), act
        assert np.array_equal(got[0][np.isinf(want)], want[np.isinf(want)].astype(dtype)), act
        ref.within(got[:, finite], np.tile(want[finite], (rows, 1)), np.abs(np.tile(want[finite], (rows, 1))) * ref.ACT_RELATIVE[dtype], dtype)
        ones = np.ones((rows, cols), dtype)
        d, _ = be.activationGrad(ones, np.tile(bias, (rows, 1)), rows, cols, dtype, act)
        d = d.onCPU(dtype).reshape(rows, cols)[0]
        nan = np.isnan(z)
        if act in ("gelu", "gelu_tanh", "silu"):
            assert np.isnan(d[nan]).all()
        limit = ref.slope(np.clip(np.where(nan, 0, z), -80, 80), act)     # flat beyond
        ref.within(d[~nan], limit[~nan], 2e-5, dtype)


def test_residual_in_place_and_overlaps_refused(be):
    import torch
    rows, inner, cols = 200, 128, 264
    rng = np.random.default_rng(5)
    a, b, _, _ = operands(rng, rows, inner, cols, np.float16)
    r = rng.standard_normal((rows, cols)).astype(np.float16)
    t = torch.from_numpy(r.copy()).cuda()
    torch.cuda.synchronize()
    be.matmulEpilogue(a, False, b, False, rows, inner, cols, np.float16, activation="silu", residual=t, out=t)
    want = be.matmulEpilogue(a, False, b, False, rows, inner, cols, np.float16, activation="silu", residual=r).onCPU(np.float16)
    be.sync()
    assert np.array_equal(t.cpu().numpy().reshape(-1), want[: rows * cols])
    buf = torch.zeros(rows * cols + inner * cols, dtype=torch.float16, device="cuda")
    bt = torch.from_numpy(b).cuda()
    at = torch.from_numpy(a).cuda()
    torch.cuda.synchronize()
    call = lambda **k: be.matmulEpilogue(at, False, bt, False, rows, inner, cols, np.float16, **k)  # noqa: E731
    with pytest.raises(ValueError, match="overlaps"):
        call(out=buf[: rows * cols], residual=buf[8: 8 + rows * cols])
    with pytest.raises(ValueError, match="overlaps"):
        call(out=buf[: rows * cols], pre=buf[: rows * cols])
    with pytest.raises(ValueError, match="overlaps"):
        be.matmulEpilogue(at, False, buf[: inner * cols], False, rows, inner, cols, np.float16, out=buf[: rows * cols])
    with pytest.raises(ValueError, match="excludes"):
        call(gradPre=buf[: rows * cols], bias=buf[:cols])
    with pytest.raises(ValueError, match="activation"):
        call(activation="tanh")
    with pytest.raises(ValueError, match="smaller"):
        call(bias=buf[: cols - 1])
    with pytest.raises(ValueError, match="type"):
        call(bias=torch.zeros(cols, dtype=torch.bfloat16, device="cuda"))


def test_unaligned_tensors(be):
    """Tensors that start off a 16-byte boundary: element accesses, the same values."""
    import torch
    rows, inner, cols = 140, 64, 264
    for dtype, tt in ((np.float16, torch.float16), (np.float32, torch.float32)):
        rng = np.random.default_rng(2)
        a, b, _, _ = operands(rng, rows, inner, cols, dtype)
        host = [a.reshape(-1), b.reshape(-1), rng.standard_normal(cols).astype(dtype), rng.standard_normal(rows * cols).astype(dtype)]
        want = be.matmulEpilogue(a, False, b, False, rows, inner, cols, dtype, activation="gelu", bias=host[2],
                                 residual=host[3]).onCPU(dtype)[: rows * cols]

        def off(x):
            t = torch.zeros(x.size + 1, dtype=tt, device="cuda")
            t[1:] = torch.from_numpy(x).cuda()
            return t[1:]

        dev = [off(x) for x in host]
        pre, out = off(np.zeros(rows * cols, dtype)), off(np.zeros(rows * cols, dtype))
        torch.cuda.synchronize()
        be.matmulEpilogue(dev[0], False, dev[1], False, rows, inner, cols, dtype, activation="gelu", bias=dev[2], residual=dev[3],
                          pre=pre, out=out)
        be.sync()
        assert np.array_equal(out.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_gradients_against_differences(be, dtype):
    """The gradient of sum(out * g) along a direction of the pre-activation, by central differences in float64."""
    rng = np.random.default_rng(11)
    rows, cols = 9, 40
    g = rng.standard_normal((rows, cols)).astype(dtype)
    pre = (rng.standard_normal((rows, cols)) * 1.5).astype(dtype)
    v = rng.standard_normal((rows, cols))
    z, g64, h = pre.astype(np.float64), g.astype(np.float64), 1e-5
    for act in ("gelu", "gelu_tanh", "silu"):
        out, _ = be.activationGrad(g, pre, rows, cols, dtype, act)
        along = float((out.onCPU(dtype)[: rows * cols].astype(np.float64).reshape(rows, cols) * v).sum())
        diff = float((g64 * (ref.activation(z + h * v, act) - ref.activation(z - h * v, act))).sum() / (2 * h))
        # each of the terms is rounded by half a step at most; 1e-8 for the difference quotient
        room = float((np.abs(g64 * v) * 1.2).sum()) * (ref.HALF_STEP[dtype] + 2e-5) + 1e-6
        assert abs(along - diff) <= room


def test_replayed_graph_and_growth_of_the_work_area(be):
    """A captured call whose work area grows during the capture, calls that outgrow it afterwards, and the replay."""
    import torch
    from honeycrisp_b200 import CUDABackend
    rng = np.random.default_rng(8)
    rows, inner, cols = 128, 2048, 128           # float32 halves: needs a work area
    a, b, _, _ = operands(rng, rows, inner, cols, np.float32)
    ad, bd = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()
    out = torch.empty(rows, cols, device="cuda")
    big = [torch.from_numpy(x).cuda() for x in operands(rng, 1024, 1024, 1024, np.float32)[:2]]
    fresh = CUDABackend(0)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    fresh.useStream(s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        fresh.matmulEpilogue(ad, False, bd, False, rows, inner, cols, np.float32, activation="gelu", out=out, mark=False)
    want = be.matmulEpilogue(a, False, b, False, rows, inner, cols, np.float32, activation="gelu").onCPU(np.float32)[: rows * cols]
    for _ in range(2):
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy().reshape(-1), want)
        fresh.matmulEpilogue(big[0], False, big[1], False, 1024, 1024, 1024, np.float32, activation="relu")
        fresh.sync()
    del g
    fresh.checkDeviceStatus()
    fresh.close()


@pytest.mark.parametrize("shape", [0, 1, 2, 3, 4, 5, 6])
@pytest.mark.parametrize("rows", [2, 3, 7, 8, 9, 15, 16, 17, 33, 131, 160 + 8, 256 + 12])
def test_warps_with_few_rows(diag, monkeypatch, rows, shape):
    """Tiles whose last 32 rows hold one to sixteen: their columns are shared among the lanes; with and without TMA, every extra, the gradient."""
    if shape:
        monkeypatch.setenv("HC_TC_SHAPE", str(shape))
    monkeypatch.setenv("HC_TC_SPLITS", "1")
    for cols in (72, 520, 517):
        for act, extras in (("gelu", (True, False, False)), ("silu", (False, True, True)), ("none", (True, True, False)), ("relu", (False, False, True))):
            forward_case(diag, rows, 136, cols, np.float16, act, *extras, tb=cols == 520)
        rng = np.random.default_rng(rows + cols)
        a, b, _, _ = operands(rng, rows, 136, cols, np.float16)
        pre = rng.standard_normal((rows, cols)).astype(np.float16)
        out = diag.matmulEpilogue(a, False, b, False, rows, 136, cols, np.float16, activation="gelu_tanh", gradPre=pre)
        d = ref.slope(pre.astype(np.float64), "gelu_tanh")
        z = a.astype(np.float64) @ b.astype(np.float64)
        ref.within(out.onCPU(np.float16)[: rows * cols], z * d, ref.product_error(a, b, np.float16) * np.abs(d) + np.abs(z) * 4e-5, np.float16)
