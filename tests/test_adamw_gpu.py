"""The AdamW step over many tensors, against its formulas in float64."""
import numpy as np
import pytest

import operator_reference as ref

pytestmark = pytest.mark.gpu

HYPER = dict(learningRate=3e-3, beta1=0.9, beta2=0.995, epsilon=1e-8, weightDecay=0.1)


@pytest.fixture(scope="module")
def be():
    from honeycrisp_b200 import CUDABackend
    b = CUDABackend(0)
    yield b
    b.checkDeviceStatus()
    b.close()


def step64(p, g, m, v, step, h):
    m = h["beta1"] * m + (1 - h["beta1"]) * g
    v = h["beta2"] * v + (1 - h["beta2"]) * g * g
    u = (m / (1 - h["beta1"] ** step)) / (np.sqrt(v / (1 - h["beta2"] ** step)) + h["epsilon"])
    return p * (1 - h["learningRate"] * h["weightDecay"]) - h["learningRate"] * u, m, v, u


def make(rng, n, pt, gt, torch, off=0):
    tt = {np.float16: torch.float16, np.float32: torch.float32}
    host = {"param": (rng.standard_normal(n) * 0.1).astype(pt), "grad": (rng.standard_normal(n) * 1e-2).astype(gt),
            "moment1": (rng.standard_normal(n) * 1e-2).astype(np.float32), "moment2": (rng.random(n) * 1e-4).astype(np.float32)}
    dev = {}
    for k, x in host.items():
        t = torch.zeros(n + off, dtype=tt[x.dtype.type], device="cuda")
        t[off:] = torch.from_numpy(x).cuda()
        dev[k] = t[off:]
    return host, dev


@pytest.mark.parametrize("pt,gt,copy", [(np.float32, np.float32, False), (np.float32, np.float16, True), (np.float16, np.float16, False),
                                        (np.float16, np.float32, False), (np.float32, np.float32, True)])
def test_many_tensors_of_odd_sizes(be, pt, gt, copy):
    import torch
    rng = np.random.default_rng(1)
    sizes = [1, 2, 3, 8, 17, 255, 256, 4095, 4096, 4097, 8192, 10001, 65536, 100003]
    made = [make(rng, n, pt, gt, torch, off=i % 3) for i, n in enumerate(sizes)]
    copies = [torch.full((n,), 9.0, dtype=torch.float16, device="cuda") if copy and i != 4 else None for i, n in enumerate(sizes)]
    plan = be.adamWPlan([dict(d, copy=c) for (_, d), c in zip(made, copies)])
    torch.cuda.synchronize()
    state = [{k: x.astype(np.float64) for k, x in h.items()} for h, _ in made]
    for step in (1, 2, 3):
        be.adamW(plan, step, **HYPER)
        be.sync()
        for s, (_, d), c in zip(state, made, copies):
            p, m, v, u = step64(s["param"], s["grad"], s["moment1"], s["moment2"], step, HYPER)
            got = {k: d[k].cpu().numpy() for k in ("param", "moment1", "moment2")}
            em = (np.abs(s["moment1"]) + np.abs(s["grad"])) * 2.0 ** -23      # factors and two roundings
            ev = v * 2.0 ** -21
            ref.within(got["moment1"], m, em, np.float32)
            ref.within(got["moment2"], v, ev, np.float32)
            bias1 = 1 - HYPER["beta1"] ** step
            room = np.sqrt(v / (1 - HYPER["beta2"] ** step)) + HYPER["epsilon"]
            eu = np.abs(u) * 2.0 ** -19 + em / bias1 / room
            ep = HYPER["learningRate"] * eu + (np.abs(s["param"]) + HYPER["learningRate"] * np.abs(u)) * 2.0 ** -22
            ref.within(got["param"], p, ep, pt)
            if c is not None:
                ref.within(c.cpu().numpy(), p, ep + np.abs(p) * ref.HALF_STEP[pt], np.float16)
            # the next step starts from what the device holds
            for k in got:
                s[k] = got[k].astype(np.float64)


def test_more_tensors_than_one_launch_takes(be):
    import torch
    rng = np.random.default_rng(2)
    n, count = 33, 1000
    flat = {k: torch.from_numpy((rng.standard_normal(n * count) * 0.01).astype(np.float32)).cuda() for k in ("param", "grad", "moment1")}
    flat["moment2"] = flat["grad"] ** 2
    before = {k: v.cpu().numpy().astype(np.float64) for k, v in flat.items()}
    plan = be.adamWPlan([{k: v[i * n: (i + 1) * n] for k, v in flat.items()} for i in range(count)])
    torch.cuda.synchronize()
    launches = be.launchCount()
    be.adamW(plan, 5, **HYPER)
    be.sync()
    assert 1 < be.launchCount() - launches <= 4
    p, m, v, _ = step64(before["param"], before["grad"], before["moment1"], before["moment2"], 5, HYPER)
    ref.within(flat["param"].cpu().numpy(), p, np.abs(p) * 2.0 ** -21 + HYPER["learningRate"] * 20 * 2.0 ** -19, np.float32)
    ref.within(flat["moment1"].cpu().numpy(), m, (np.abs(before["moment1"]) + np.abs(before["grad"])) * 2.0 ** -23, np.float32)


def test_neighbours_and_empty_tensors_are_left_alone(be):
    import torch
    buf = {k: torch.full((100,), 0.5, device="cuda") for k in ("param", "grad", "moment1", "moment2")}
    plan = be.adamWPlan([{k: v[7:40] for k, v in buf.items()}, {k: v[50:50] for k, v in buf.items()}])
    torch.cuda.synchronize()
    be.adamW(plan, 1)
    be.sync()
    for k in ("param", "moment1", "moment2"):
        x = buf[k].cpu().numpy()
        assert (x[:7] == 0.5).all() and (x[40:] == 0.5).all()
        # 0.9 * 0.5 + 0.1 * 0.5 leaves the first moment where it is
        assert (x[7:40] != 0.5).all() or k == "moment1"
    assert (buf["grad"].cpu().numpy() == 0.5).all()


def test_no_gradient_leaves_decay_alone_and_nan_stays_where_it_is(be):
    import torch
    p = torch.full((64,), 2.0, device="cuda")
    g, m, v = (torch.zeros(64, device="cuda") for _ in range(3))
    g[3] = float("nan")
    plan = be.adamWPlan([dict(param=p, grad=g, moment1=m, moment2=v)])
    torch.cuda.synchronize()
    be.adamW(plan, 1, learningRate=0.5, weightDecay=0.5)
    be.sync()
    x = p.cpu().numpy()
    assert np.isnan(x[3]) and (np.delete(x, 3) == 1.5).all()


def test_refusals(be):
    import torch
    t = [torch.zeros(16, device="cuda") for _ in range(4)]
    plan = be.adamWPlan([dict(param=t[0], grad=t[1], moment1=t[2], moment2=t[3])])
    for bad, what in ((dict(step=0), "step"), (dict(step=1, beta1=1.0), "beta"), (dict(step=1, epsilon=-1.0), "epsilon")):
        with pytest.raises(ValueError, match=what):
            be.adamW(plan, **bad)
    with pytest.raises(ValueError, match="overlap"):
        be.adamWPlan([dict(param=t[0], grad=t[1], moment1=t[2], moment2=t[2])])
    plan._table[0].moment2 = plan._table[0].moment1          # past the plan's own check, the library's
    with pytest.raises(ValueError, match="overlap"):
        be.adamW(plan, 1)
    with pytest.raises(ValueError, match="smaller"):
        be.adamWPlan([dict(param=t[0], grad=t[1][:5], moment1=t[2], moment2=t[3])])
    with pytest.raises(ValueError, match="type"):
        be.adamWPlan([dict(param=t[0], grad=t[1], moment1=t[2].half(), moment2=t[3])])
    from honeycrisp_b200 import NotImplementedByBackend
    with pytest.raises(NotImplementedByBackend):
        be.adamWPlan([dict(param=t[0].bfloat16(), grad=t[1], moment1=t[2], moment2=t[3])])
