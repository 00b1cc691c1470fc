"""The operators together, as a feed-forward block's training step uses them, against float64 automatic differentiation."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

# Relative Frobenius room.  float16: every tensor a result passes through is rounded by 2^-11 of its values at most; a block's
# gradient passes through seven of them (n, pre, h, out's gradient product, dPre, dn, dx), each weighted by factors of
# norm about one or two.  float32: products of 1e-6 each.
ROOM = {np.float16: 16 * 2.0 ** -11, np.float32: 2e-5}


@pytest.fixture(scope="module")
def be():
    from honeycrisp_b200 import CUDABackend
    b = CUDABackend(0)
    yield b
    b.checkDeviceStatus()
    b.close()


def rel(got, want):
    want = np.asarray(want, np.float64).reshape(-1)
    return float(np.linalg.norm(np.asarray(got).astype(np.float64).reshape(-1)[: want.size] - want) / np.linalg.norm(want))


def act64(z, name):
    import torch
    return {"gelu": lambda: z * torch.special.erfc(-z / 2 ** 0.5) / 2, "silu": lambda: z * torch.sigmoid(z), "relu": lambda: z.clamp(min=0),
            "gelu_tanh": lambda: z * torch.sigmoid(1.5957691216057308 * (z + 0.044715 * z ** 3))}[name]()


def block64(x, params, name):
    nw, nb, uw, ub, dw, db = params
    m = x.mean(1, keepdim=True)
    h = (x - m) / ((x - m) ** 2).mean(1, keepdim=True).add(1e-5).sqrt()
    return x + act64((h * nw + nb) @ uw + ub, name) @ dw + db


def parameters_of(be, block):
    import torch
    out = []
    for p, _, n, t in block.parameters():
        out.append(torch.from_numpy(p.onCPU(t.numpy)[:n].astype(np.float64)))
    w, h = block.width, block.hidden
    shapes = [(w,), (w,), (w, h), (h,), (h, w), (w,)]
    return [p.reshape(s).requires_grad_() for p, s in zip(out, shapes)]


@pytest.mark.parametrize("dtype,name,rows,width,hidden", [(np.float16, "gelu", 192, 256, 520), (np.float32, "gelu_tanh", 100, 96, 264),
                                                          (np.float16, "silu", 3, 64, 256), (np.float32, "relu", 257, 130, 67)])
def test_training_step_of_a_block(be, dtype, name, rows, width, hidden):
    """Forward, backward and two AdamW steps: float16 computes on float32 master weights, cast on use."""
    import torch
    from honeycrisp_b200 import AdamW, FeedForward
    rng = np.random.default_rng(rows)
    block = FeedForward(be, width, hidden, activation=name, dtype=np.float32, castParams=dtype if dtype == np.float16 else None, seed=3)
    block.norm.weight = be.collection((1 + 0.1 * rng.standard_normal(width)).astype(np.float32), np.float32)
    block.norm.bias = be.collection((0.1 * rng.standard_normal(width)).astype(np.float32), np.float32)
    block.up.bias = be.collection((0.1 * rng.standard_normal(hidden)).astype(np.float32), np.float32)
    block.down.bias = be.collection((0.1 * rng.standard_normal(width)).astype(np.float32), np.float32)
    optimiser = AdamW(be, [block], learningRate=1e-2, weightDecay=0.1)
    for step in (1, 2):
        x = rng.standard_normal((rows, width)).astype(dtype)
        g = rng.standard_normal((rows, width)).astype(dtype)
        params = parameters_of(be, block)
        x64 = torch.from_numpy(x.astype(np.float64)).requires_grad_()
        want = block64(x64, params, name)
        want.backward(torch.from_numpy(g.astype(np.float64)))
        out, saved = block(be.collection(x, dtype), rows)
        dx = block.backward(be.collection(g, dtype), saved)
        assert rel(out.onCPU(dtype), want.detach().numpy()) < ROOM[dtype]
        assert rel(dx.onCPU(dtype), x64.grad.numpy()) < ROOM[dtype]
        grads = []
        for (p, got, n, t), p64 in zip(block.parameters(), params):
            got = got.onCPU(t.numpy)[:n].astype(np.float64)
            assert rel(got, p64.grad.numpy()) < ROOM[dtype]
            grads.append(got)
        before = [p.detach().numpy().reshape(-1).copy() for p in params]
        moments = [tuple(v.onCPU(np.float32)[: b.size].astype(np.float64) for v in mv) for mv, b in zip(optimiser.moments, before)] or [(0 * b, 0 * b) for b in before]
        optimiser.step()
        for (p, _, n, t), b, gr, (m, v) in zip(block.parameters(), before, grads, moments):
            m, v = 0.9 * m + 0.1 * gr, 0.999 * v + 0.001 * gr * gr
            u = m / (1 - 0.9 ** step) / (np.sqrt(v / (1 - 0.999 ** step)) + 1e-8)
            w = b * (1 - 1e-3) - 1e-2 * u
            assert np.abs(p.onCPU(t.numpy)[:n] - w).max() <= 2.0 ** -20 * (np.abs(w).max() + 1e-2 * np.abs(u).max())
        optimiser.zeroGrad()


def test_layer_with_activation_alone(be):
    """A Linear layer whose activation has no product behind it: the gradient through it brings the bias's along, and gradients accumulate."""
    import torch
    from honeycrisp_b200 import Linear
    rng = np.random.default_rng(0)
    layer = Linear(be, 72, 136, activation="gelu", seed=1)
    x, g = (rng.standard_normal(s).astype(np.float32) for s in ((2, 33, 72), (66, 136)))
    out, shape, pre = layer.forwardKeepingPre(x, [2, 33, 72])
    assert shape == [2, 33, 136] and np.array_equal(out.onCPU(), layer(x, [2, 33, 72])[0].onCPU())
    w = torch.from_numpy(layer.weight.onCPU(np.float32)[: 72 * 136].reshape(72, 136).astype(np.float64)).requires_grad_()
    b = torch.zeros(136, dtype=torch.float64, requires_grad=True)
    x64 = torch.from_numpy(x.reshape(66, 72).astype(np.float64)).requires_grad_()
    y = act64(x64 @ w + b, "gelu")
    y.backward(torch.from_numpy(g.astype(np.float64)))
    assert rel(out.onCPU(np.float32), y.detach().numpy()) < 1e-5
    for times in (1, 2):
        dx = layer.backward(x, [2, 33, 72], g, pre=pre)
        assert rel(dx.onCPU(np.float32), x64.grad.numpy()) < 1e-5
        assert rel(layer.weightGrad.onCPU(np.float32), times * w.grad.numpy()) < 1e-5
        assert rel(layer.biasGrad.onCPU(np.float32), times * b.grad.numpy()) < 1e-5
    with pytest.raises(ValueError, match="pre"):
        layer.backward(x, [2, 33, 72], g)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_experts_forward_and_backward(be, dtype):
    from honeycrisp_b200 import AdamW, Experts
    rng = np.random.default_rng(2)
    groups, n_in, n_out, rows = 5, 136, 72, 300
    ends = [0, 120, 120, 200, 280, 290]
    experts = Experts(be, groups, n_in, n_out, dtype, seed=4)
    w = experts.weight.onCPU(dtype).reshape(groups, n_in, n_out).astype(np.float64)
    x, g = rng.standard_normal((rows, n_in)).astype(dtype), rng.standard_normal((rows, n_out)).astype(dtype)
    offsets = be.collection(np.array(ends), np.int64)
    xd, gd = be.collection(x, dtype), be.collection(g, dtype)
    out, dx = np.zeros((rows, n_out)), np.zeros((rows, n_in))
    dw = np.zeros_like(w)
    for i in range(groups):
        s = slice(ends[i], ends[i + 1])
        out[s] = x[s].astype(np.float64) @ w[i]
        dx[s] = g[s].astype(np.float64) @ w[i].T
        dw[i] = x[s].astype(np.float64).T @ g[s].astype(np.float64)
    assert rel(experts(xd, offsets, rows).onCPU(dtype), out) < ROOM[dtype]
    got = experts.backward(xd, offsets, rows, gd)
    assert rel(got.onCPU(dtype), dx) < ROOM[dtype]
    assert rel(experts.weightGrad.onCPU(dtype), dw) < ROOM[dtype]
    assert not got.onCPU(dtype).reshape(rows, n_in)[290:].any()
    AdamW(be, [experts]).step()
    after = experts.weight.onCPU(dtype).reshape(w.shape).astype(np.float64)
    # No rows, no gradient, decay alone: the factor 1 - 1e-5 is rounded to float32 (2^-25 off), the product rounded (2^-24), then the
    # parameter to its type.
    assert (np.abs(after[1] - w[1] * (1 - 1e-5)) <= np.abs(w[1]) * (2.0 ** -25 + 2.0 ** -24 + (2.0 ** -11 if dtype == np.float16 else 0))).all()
    assert (after[[0, 2, 3, 4]] != w[[0, 2, 3, 4]]).mean() > 0.9


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_captured_training_step(be, dtype):
    """Every operator of a step in one graph on a fresh context (its work area grows during the capture), replayed on new inputs: the
    bits of the same calls made one by one."""
    import torch
    from honeycrisp_b200 import CUDABackend
    tt = {np.float16: torch.float16, np.float32: torch.float32}[dtype]
    rows, width, hidden, groups = 200, 136, 264, 3
    gen = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *s, t=tt, scale=1.0: (torch.randn(*s, generator=gen, device="cuda") * scale).to(t)  # noqa: E731
    buf = dict(x=new(rows, width), g=new(rows, width), nw=new(width, t=torch.float32), nb=new(width, t=torch.float32), uw=new(width, hidden, scale=0.1),
               ub=new(hidden), dw=new(hidden, width, scale=0.1), db=new(width), ew=new(groups, width, width, scale=0.1))
    buf["offsets"] = torch.tensor([0, 50, 51, 190], device="cuda")

    def tensors():
        z = lambda *s, t=tt: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
        f = torch.float32
        return dict(n=z(rows, width), mean=z(rows, t=f), rstd=z(rows, t=f), h=z(rows, hidden), pre=z(rows, hidden), out=z(rows, width),
                    dpre=z(rows, hidden), gpre=z(rows, hidden), ubg=z(hidden, t=f), uwg=z(width, hidden), dwg=z(hidden, width), dn=z(rows, width),
                    dx=z(rows, width), nwg=z(width, t=f), nbg=z(width, t=f), eo=z(rows, width), ewg=z(groups, width, width),
                    m=z(width, hidden, t=f), v=z(width, hidden, t=f))

    def calls(b, r, plan):
        dt, k = dtype, dict(mark=False)
        wrap = lambda t: b.wrap(t.data_ptr(), t.numel() * t.element_size())  # noqa: E731
        b.layerNorm(buf["x"], buf["nw"], buf["nb"], rows, width, dt, out=r["n"], mean=r["mean"], rstd=r["rstd"], **k)
        b.matmulEpilogue(r["n"], False, buf["uw"], False, rows, width, hidden, dt, activation="gelu", bias=buf["ub"], pre=r["pre"], out=r["h"], **k)
        b.matmulEpilogue(r["h"], False, buf["dw"], False, rows, hidden, width, dt, bias=buf["db"], residual=buf["x"], out=r["out"], **k)
        b.matmulEpilogue(buf["g"], False, buf["dw"], True, rows, width, hidden, dt, activation="gelu", gradPre=r["pre"], out=r["dpre"], **k)
        b.activationGrad(r["h"], r["pre"], rows, hidden, dt, "silu", out=r["gpre"], biasGrad=r["ubg"], **k)
        b.matmul(r["n"], True, r["dpre"], False, False, width, rows, hidden, dt, out=wrap(r["uwg"]), **k)
        b.matmul(r["h"], True, buf["g"], False, False, hidden, rows, width, dt, out=wrap(r["dwg"]), **k)
        b.matmul(r["dpre"], False, buf["uw"], True, False, rows, hidden, width, dt, out=wrap(r["dn"]), **k)
        b.layerNormGrad(r["dn"], buf["x"], buf["nw"], r["mean"], r["rstd"], rows, width, dt, out=r["dx"], weightGrad=r["nwg"], biasGrad=r["nbg"], **k)
        b.groupedMatmul(groups, buf["offsets"], buf["x"], buf["ew"], False, rows, width, width, dt, out=r["eo"], **k)
        b.groupedMatmulWeightGrad(groups, buf["offsets"], buf["x"], buf["g"], rows, width, width, dt, out=r["ewg"], **k)
        b.adamW(plan, 3, mark=False)

    one, other = tensors(), tensors()
    weights = [buf["uw"].clone(), buf["uw"].clone()]
    plans = [be.adamWPlan([dict(param=w, grad=r["uwg"], moment1=r["m"], moment2=r["v"])]) for w, r in zip(weights, (one, other))]
    fresh = CUDABackend(0)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    fresh.useStream(s.cuda_stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        calls(fresh, one, plans[0])
    for _ in range(3):
        buf["x"].copy_(new(rows, width))
        buf["g"].copy_(new(rows, width))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        calls(be, other, plans[1])
        be.sync()
        for name in one:
            assert torch.equal(one[name], other[name]), name
        assert torch.equal(*weights)
    del graph
    fresh.checkDeviceStatus()
    fresh.close()
