"""Products grouped by expert, forward and weight gradient, against plain products in float64."""
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


def check_forward(be, ends, total, inner, cols, dtype, trans_b, seed=0, first=0):
    import torch
    rng = np.random.default_rng(seed + total + inner + cols)
    groups = len(ends) - 1
    a = rng.standard_normal((total, inner)).astype(dtype)
    b = (rng.standard_normal((groups, inner, cols)) / np.sqrt(max(1, inner))).astype(dtype)
    stored = np.ascontiguousarray(np.swapaxes(b, 1, 2)) if trans_b else b
    out = torch.full((total, cols), 0.25, dtype={np.float16: torch.float16, np.float32: torch.float32}[dtype], device="cuda")
    # what lies outside the groups must reach nothing
    poisoned = a.copy()
    poisoned[: ends[0]] = np.nan
    poisoned[ends[-1]:] = np.inf
    torch.cuda.synchronize()
    be.groupedMatmul(groups, np.asarray(ends, np.int64), poisoned, stored, trans_b, total, inner, cols, dtype, out=out)
    be.sync()
    got = out.cpu().numpy()
    assert (got[: ends[0]] == 0.25).all() and (got[ends[-1]:] == 0.25).all()
    for g in range(groups):
        s, e = ends[g], ends[g + 1]
        if e > s:
            ref.within(got[s:e], a[s:e].astype(np.float64) @ b[g].astype(np.float64), ref.product_error(a[s:e], b[g], dtype), dtype)


def check_weight_grad(be, ends, total, rows, cols, dtype, seed=0):
    rng = np.random.default_rng(seed + total + rows + cols)
    groups = len(ends) - 1
    a = rng.standard_normal((total, rows)).astype(dtype)
    b = rng.standard_normal((total, cols)).astype(dtype)
    for x in (a, b):
        x[: ends[0]] = np.nan
        x[ends[-1]:] = np.inf
    got = be.groupedMatmulWeightGrad(groups, np.asarray(ends, np.int64), a, b, total, rows, cols, dtype).onCPU(dtype)
    got = got[: groups * rows * cols].reshape(groups, rows, cols)
    for g in range(groups):
        s, e = ends[g], ends[g + 1]
        at, bt = np.ascontiguousarray(a[s:e].T), b[s:e]
        if e == s:
            assert not got[g].any()
        else:
            ref.within(got[g], at.astype(np.float64) @ bt.astype(np.float64), ref.product_error(at, bt, dtype), dtype)


CASES = [  # offsets, total rows, inner, cols
    ([0, 1], 1, 8, 8),
    ([0, 3, 3, 5], 5, 16, 24),
    ([0, 0, 0], 4, 32, 16),
    ([2, 40, 41, 90], 100, 64, 136),
    ([0, 300, 301, 301, 700], 700, 128, 264),
    ([0, 129, 385, 640], 641, 200, 520),
    ([0, 31, 63, 127, 255, 256], 256, 1000, 72),
    ([0, 77, 150], 150, 33, 41),
    ([0, 5, 9], 9, 7, 1),
    ([0, 1000], 1000, 512, 1032),
    ([0, 700, 1500], 1503, 96, 2056),
    (list(range(0, 260, 4)), 256, 128, 256),
]


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("trans_b", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_forward(be, case, trans_b, dtype):
    ends, total, inner, cols = CASES[case]
    check_forward(be, ends, total, inner, cols, dtype, trans_b)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_weight_gradient(be, case, dtype):
    ends, total, rows, cols = CASES[case]
    check_weight_grad(be, ends, total, rows, cols, dtype)


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_many_groups(be, dtype):
    """More groups than the set-up kernel takes in one round, most of them empty or of one row."""
    rng = np.random.default_rng(1)
    sizes = rng.integers(0, 3, 2500)
    ends = np.concatenate([[0], np.cumsum(sizes)]).tolist()
    check_forward(be, ends, ends[-1], 16, 24, dtype, False)
    check_weight_grad(be, ends, ends[-1], 16, 24, dtype)


def test_empty_lengths(be):
    import torch
    out = torch.full((6, 4), 2.0, device="cuda")
    torch.cuda.synchronize()
    be.groupedMatmul(2, np.array([1, 3, 5], np.int64), np.zeros((6, 0), np.float32), np.zeros((2, 0, 4), np.float32), False, 6, 0, 4,
                     np.float32, out=out)
    be.sync()
    assert out.cpu().numpy().tolist() == [[2.0] * 4] + [[0.0] * 4] * 4 + [[2.0] * 4]
    none = np.zeros(1, np.int64)
    be.groupedMatmul(0, none, np.zeros((6, 4), np.float32), np.zeros((0,), np.float32), False, 6, 4, 4, np.float32)
    got = be.groupedMatmulWeightGrad(3, np.zeros(4, np.int64), np.zeros((0, 4), np.float16), np.zeros((0, 8), np.float16), 0, 4, 8, np.float16)
    assert not got.onCPU(np.float16)[:96].any()


def test_offsets_out_of_range_stay_in_range(be):
    """Offsets that leave the rows or run backwards are clamped: what is written is what the clamped offsets say."""
    rng = np.random.default_rng(4)
    total, inner, cols = 300, 64, 72
    a = rng.standard_normal((total, inner)).astype(np.float16)
    b = rng.standard_normal((4, inner, cols)).astype(np.float16)
    bad = np.array([-50, 100, 40, 10 ** 12, 200], np.int64)
    good = np.array([0, 100, 100, 300, 300], np.int64)
    got = [be.groupedMatmul(4, o, a, b, False, total, inner, cols, np.float16).onCPU(np.float16) for o in (bad, good)]
    assert np.array_equal(*got)
    c = rng.standard_normal((total, cols)).astype(np.float16)
    got = [be.groupedMatmulWeightGrad(4, o, a, c, total, inner, cols, np.float16).onCPU(np.float16) for o in (bad, good)]
    assert np.array_equal(*got)


def test_captured_call_follows_new_offsets(be):
    import torch
    from honeycrisp_b200 import CUDABackend
    rng = np.random.default_rng(9)
    total, inner, cols, groups = 400, 128, 264, 3
    a = torch.from_numpy(rng.standard_normal((total, inner)).astype(np.float16)).cuda()
    b = torch.from_numpy(rng.standard_normal((groups, inner, cols)).astype(np.float16)).cuda()
    c = torch.from_numpy(rng.standard_normal((total, cols)).astype(np.float16)).cuda()
    offsets = torch.tensor([0, 100, 250, 400]).cuda()
    out, dw = torch.zeros(total, cols, dtype=torch.float16, device="cuda"), torch.zeros(groups, inner, cols, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    fresh = CUDABackend(0)
    s = torch.cuda.Stream()
    fresh.useStream(s.cuda_stream)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        fresh.groupedMatmul(groups, offsets, a, b, False, total, inner, cols, np.float16, out=out, mark=False)
        fresh.groupedMatmulWeightGrad(groups, offsets, a, c, total, inner, cols, np.float16, out=dw, mark=False)
    for ends in ([0, 100, 250, 400], [0, 0, 399, 400], [10, 11, 12, 300]):
        offsets.copy_(torch.tensor(ends))
        out.fill_(0.5)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = torch.full_like(out, 0.5)
        torch.cuda.synchronize()
        be.groupedMatmul(groups, offsets, a, b, False, total, inner, cols, np.float16, out=want)
        wdw = be.groupedMatmulWeightGrad(groups, offsets, a, c, total, inner, cols, np.float16)
        be.sync()
        assert torch.equal(out, want)
        assert np.array_equal(dw.cpu().numpy().reshape(-1), wdw.onCPU(np.float16)[: dw.numel()])
    del g
    fresh.checkDeviceStatus()
    fresh.close()


def test_refusals(be):
    import torch
    a = torch.zeros(8, 8, dtype=torch.float16, device="cuda")
    b = torch.zeros(2, 8, 8, dtype=torch.float16, device="cuda")
    o = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="type"):
        be.groupedMatmul(2, o.int(), a, b, False, 8, 8, 8, np.float16)
    with pytest.raises(ValueError, match="smaller"):
        be.groupedMatmul(2, o[:2], a, b, False, 8, 8, 8, np.float16)
    with pytest.raises(ValueError, match="smaller"):
        be.groupedMatmul(3, torch.zeros(4, dtype=torch.int64, device="cuda"), a, b, False, 8, 8, 8, np.float16)
    with pytest.raises(ValueError, match="overlaps"):
        be.groupedMatmul(2, o, a, b, False, 8, 8, 8, np.float16, out=a)
    with pytest.raises(ValueError, match="negative"):
        be.groupedMatmul(-1, o, a, b, False, 8, 8, 8, np.float16, out=torch.zeros_like(a))
