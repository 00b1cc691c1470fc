"""The feed-forward operators on tensors of more than 2^31 elements.  A small pattern is repeated through the tensor, so every repetition of
the result has to carry the first one's bits (the other files compare small results with 64 bits)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF = np.float16


@pytest.fixture(scope="module")
def be():
    import torch
    from honeycrisp_b200 import CUDABackend
    b = CUDABackend(0)
    yield b
    b.checkDeviceStatus()
    b.close()
    torch.cuda.empty_cache()


def randn(*shape, seed=0, scale=1.0, dtype=None):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype or torch.float16)


def repeats(t, axis, period):
    """Whole periods of `t` along `axis` all equal the first; bits, so that nothing is lost on signs of zero."""
    import torch
    bits = t.view(torch.int16 if t.element_size() == 2 else torch.int32)
    n = t.shape[axis] // period
    first = bits.narrow(axis, 0, period)
    return all(torch.equal(bits.narrow(axis, i * period, period), first) for i in (1, n // 2, n - 2, n - 1)) and bool(
        (bits.narrow(axis, 0, n * period).unflatten(axis, (n, period)) == first.unsqueeze(axis)).all())


@pytest.mark.parametrize("cols", [4096, 4099])
def test_rows(be, cols):
    import torch
    period, times = 64, 8200
    rows = period * times
    assert rows * cols > 2 ** 31
    x0, g0 = randn(period, cols, seed=1), randn(period, cols, seed=2)
    x = x0.repeat(times, 1)
    w, b = randn(cols, seed=3, dtype=torch.float32), randn(cols, seed=4, dtype=torch.float32)
    out = torch.zeros_like(x)
    mean, rstd = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    be.layerNorm(x, w, b, rows, cols, HALF, out=out, mean=mean, rstd=rstd)
    be.sync()
    assert repeats(out, 0, period) and repeats(mean, 0, period) and repeats(rstd, 0, period)
    h = (x0.double() - x0.double().mean(1, keepdim=True)) / (x0.double().var(1, unbiased=False, keepdim=True) + 1e-5).sqrt()
    want = h * w + b
    # half a step of float16, and of float32 in each operation of sums of a few thousand values of about one
    assert bool(((out[:period] - want).abs() <= want.abs() * 2.0 ** -11 + (h * w).abs() * 2.0 ** -19 + 2.0 ** -18).all())
    g = g0.repeat(times, 1)
    torch.cuda.synchronize()
    be.layerNormGrad(g, x, w, mean, rstd, rows, cols, HALF, out=out, weightGrad=False, biasGrad=False)
    be.sync()
    assert repeats(out, 0, period) and bool(out[:period].any())
    be.activationGrad(g, x, rows, cols, HALF, "gelu", out=out, biasGrad=False)
    be.sync()
    assert repeats(out, 0, period) and bool(out[:period].any())
    # a gradient that is zero but for the last rows: sums of that many values
    g[:-period] = 0
    torch.cuda.synchronize()
    sums = [torch.zeros(cols, device="cuda") for _ in range(3)]
    be.layerNormGrad(g, x, w, mean, rstd, rows, cols, HALF, out=False, weightGrad=sums[0], biasGrad=sums[1])
    be.activationGrad(g, x, rows, cols, HALF, "none", out=out, biasGrad=sums[2])
    be.sync()
    gd = g0.double()
    room = gd.abs().sum(0) * period * 2.0 ** -23
    assert bool(((sums[1] - gd.sum(0)).abs() <= room).all()) and bool(((sums[2] - gd.sum(0)).abs() <= room).all())
    assert bool(((sums[0] - (gd * h).sum(0)).abs() <= (gd * h).abs().sum(0) * period * 2.0 ** -23 + gd.abs().sum(0) * 2.0 ** -19).all())


@pytest.mark.parametrize("cols", [256, 257])
def test_product_with_a_long_result(be, cols):
    import torch
    period, times, inner = 256, 32800, 64
    rows = period * times
    assert rows * cols > 2 ** 31
    a = randn(period, inner, seed=1).repeat(times, 1)
    b, bias = randn(inner, cols, seed=2, scale=0.1), randn(cols, seed=3)
    res = randn(period, cols, seed=4).repeat(times, 1)
    out, pre = torch.zeros_like(res), torch.zeros_like(res)
    torch.cuda.synchronize()
    be.matmulEpilogue(a, False, b, False, rows, inner, cols, HALF, activation="gelu", bias=bias, residual=res, pre=pre, out=out)
    be.sync()
    assert repeats(out, 0, period) and repeats(pre, 0, period) and bool(out[:period].any())
    z = a[:period].double() @ b.double() + bias
    assert bool(((pre[-period:] - z).abs() <= z.abs() * 2.0 ** -11 + (a[:period].double().abs() @ b.double().abs()) * inner * 2.0 ** -23 + 2.0 ** -22).all())
    be.matmulEpilogue(a, False, b, False, rows, inner, cols, HALF, activation="silu", gradPre=pre, out=out)
    be.sync()
    assert repeats(out, 0, period) and bool(out[:period].any())


@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("rows", [1, 4, 16])
@pytest.mark.parametrize("extra", [0, 1])
def test_product_with_a_large_matrix(be, rows, trans_b, extra):
    import torch
    period, inner = 512, 131072 + extra   # extra: rows off 16-byte boundaries
    times = 33
    cols = period * times
    assert inner * cols > 2 ** 31
    a = randn(rows, inner, seed=1)
    b = randn(period, inner, seed=2, scale=0.01).repeat(times, 1) if trans_b else randn(inner, period, seed=2, scale=0.01).repeat(1, times)
    out = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    be.matmulEpilogue(a, False, b, trans_b, rows, inner, cols, HALF, out=out)
    be.sync()
    assert repeats(out, 1, period)
    first = b[:period].t() if trans_b else b[:, :period]
    want = a.double() @ first.double()
    room = want.abs() * 2.0 ** -11 + (a.double().abs() @ first.double().abs()) * 2.0 ** -15   # sums of some thousands of float32 each
    assert bool(((out[:, :period] - want).abs() <= room).all())


@pytest.mark.parametrize("inner,cols", [(64, 4096), (4096, 64), (4099, 33)])
def test_groups_of_many_rows(be, inner, cols):
    import torch
    period, times = 64, 8200
    total = period * times
    a = randn(period, inner, seed=1).repeat(times, 1)
    b = randn(1, inner, cols, seed=2, scale=0.05).repeat(3, 1, 1)
    offsets = torch.tensor([0, period, total - period, total], device="cuda")
    out = torch.zeros(total, cols, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    be.groupedMatmul(3, offsets, a, b, False, total, inner, cols, HALF, out=out)
    be.sync()
    assert repeats(out, 0, period)
    want = a[:period].double() @ b[0].double()
    assert bool(((out[:period] - want).abs() <= want.abs() * 2.0 ** -11 + (a[:period].double().abs() @ b[0].double().abs()) * inner * 2.0 ** -24).all())
    # weight gradient: the first and the last group's rows are alike
    if inner > cols:
        grad = randn(period, cols, seed=3).repeat(times, 1)
        dw = torch.zeros(3, inner, cols, dtype=torch.float16, device="cuda")
        torch.cuda.synchronize()
        be.groupedMatmulWeightGrad(3, offsets, a, grad, total, inner, cols, HALF, out=dw)
        be.sync()
        assert torch.equal(dw[0], dw[2])
        want = a[:period].double().t() @ grad[:period].double()
        assert bool(((dw[2] - want).abs() <= want.abs() * 2.0 ** -11 + (a[:period].double().abs().t() @ grad[:period].double().abs()) * period * 2.0 ** -24).all())


@pytest.mark.parametrize("cols", [4224, 4225])
@pytest.mark.parametrize("each", [4, 32])
def test_large_matrices_of_groups(be, cols, each):
    import torch
    groups, inner = 64, 8192
    total = groups * each
    assert groups * inner * cols > 2 ** 31
    a = randn(each, inner, seed=1).repeat(groups, 1)
    b = randn(1, inner, cols, seed=2, scale=0.05).repeat(groups, 1, 1)
    offsets = torch.arange(groups + 1, device="cuda") * each
    out = torch.zeros(total, cols, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    be.groupedMatmul(groups, offsets, a, b, False, total, inner, cols, HALF, out=out)
    be.sync()
    assert repeats(out, 0, each)
    want = a[:each].double() @ b[0].double()
    assert bool(((out[:each] - want).abs() <= want.abs() * 2.0 ** -11 + (a[:each].double().abs() @ b[0].double().abs()) * 2.0 ** -17).all())
    b.zero_()   # now the weights' gradient
    torch.cuda.synchronize()
    be.groupedMatmulWeightGrad(groups, offsets, a, out, total, inner, cols, HALF, out=b)
    be.sync()
    assert repeats(b.view(groups * inner, cols), 0, inner) and bool(b[0].any())


def test_a_large_parameter(be):
    import torch
    period, times = 4099, 524000
    n = period * times
    assert n > 2 ** 31
    pattern = randn(period, seed=1)
    p, g = pattern.repeat(times), randn(period, seed=2).repeat(times)
    m, v = (torch.zeros(n, device="cuda") for _ in range(2))
    plan = be.adamWPlan([dict(param=p, grad=g, moment1=m, moment2=v)])
    torch.cuda.synchronize()
    be.adamW(plan, 1, learningRate=0.1)
    be.sync()
    for t in (p, m, v):
        assert repeats(t, 0, period)
    assert not torch.equal(p[:period], pattern) and torch.equal(m[:period], (g[:period].float() * np.float32(1 - 0.9)))
