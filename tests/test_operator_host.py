"""What the host refuses before anything reaches a device: the C entry points without a context, and the checks of the Python face."""
import ctypes

import numpy as np
import pytest

from honeycrisp_b200 import _lib as L
from honeycrisp_b200 import backend as B


def test_entry_points_without_a_context():
    lib = L.load()
    ep = L.Epilogue(0, None, None, None, None)
    bad = L.HC_ERR_INVALID_ARGUMENT
    assert lib.hc_matmul_epilogue(None, L.HC_F16, None, 0, None, 0, 1, 1, 1, ctypes.byref(ep), None) == bad
    assert lib.hc_activation_grad(None, L.HC_F16, 0, None, None, 1, 1, None, None) == bad
    assert lib.hc_layer_norm(None, L.HC_F16, L.HC_F32, None, None, None, 1, 1, 1e-5, None, None, None) == bad
    assert lib.hc_layer_norm_grad(None, L.HC_F16, L.HC_F32, None, None, None, None, None, 1, 1, None, None, None) == bad
    assert lib.hc_grouped_matmul(None, L.HC_F16, 1, None, None, None, 0, 1, 1, 1, None) == bad
    assert lib.hc_grouped_matmul_weight_grad(None, L.HC_F16, 1, None, None, None, 1, 1, 1, None) == bad
    assert lib.hc_adamw(None, None, 0, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0) == bad


class Recorder:
    """A library whose calls succeed and are written down."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return L.HC_OK
        return call


@pytest.fixture
def be():
    b = B.CUDABackend.__new__(B.CUDABackend)
    b._lib, b._ctx, b.device = Recorder(), 1, 0
    yield b
    b._ctx = None


def data(be, elements, size=2):
    return B.CUDAData(be, 256, elements * size, owns=False)


def called(be, name):
    return [a for n, a in be._lib.calls if n == name]


def test_epilogue_passes_what_it_was_given(be):
    a, b, bias, res, pre, out = data(be, 12), data(be, 20), data(be, 5), data(be, 15), data(be, 15), data(be, 15)
    assert be.matmulEpilogue(a, False, b, True, 3, 4, 5, "float16", activation="silu", bias=bias, residual=res, pre=pre, out=out, mark=False) is out
    (args,) = called(be, "hc_matmul_epilogue")
    assert args[1] == L.HC_F16 and args[3] == 0 and args[5] == 1 and args[6:9] == (3, 4, 5)
    assert out._inputs[2] is bias and out._inputs[3] is res


@pytest.mark.parametrize("change,error", [
    (dict(bias=4), "bias is smaller"), (dict(residual=14), "residual is smaller"), (dict(pre=14), "pre is smaller"),
    (dict(gradPre=14), "gradPre is smaller"), (dict(out=14), "out is smaller"), (dict(activation="swish"), "unknown activation")])
def test_epilogue_refuses(be, change, error):
    change = {k: data(be, v) if isinstance(v, int) else v for k, v in change.items()}
    change.setdefault("out", data(be, 15))
    with pytest.raises(ValueError, match=error):
        be.matmulEpilogue(data(be, 12), False, data(be, 20), False, 3, 4, 5, np.float16, **change)
    with pytest.raises(ValueError, match="operand a"):
        be.matmulEpilogue(data(be, 11), False, data(be, 20), False, 3, 4, 5, np.float16, out=data(be, 15))
    assert not called(be, "hc_matmul_epilogue")


def test_types_are_checked(be):
    import torch
    out = data(be, 16)
    with pytest.raises(ValueError, match="type"):
        be.activationGrad(np.zeros(16, np.float32), data(be, 16), 4, 4, np.float16, "gelu", out=out)
    with pytest.raises(ValueError, match="lies on"):
        be.activationGrad(torch.zeros(16, dtype=torch.float16), data(be, 16), 4, 4, np.float16, "gelu", out=out)
    with pytest.raises(ValueError, match="type"):
        be.activationGrad(torch.zeros(16, dtype=torch.bfloat16), data(be, 16), 4, 4, np.float16, "gelu", out=out)
    with pytest.raises(TypeError, match="device"):
        be.activationGrad(data(be, 16), data(be, 16), 4, 4, np.float16, "gelu", out=np.zeros(16, np.float16))
    for dtype in (np.int64, B.DType.int64):
        with pytest.raises(B.NotImplementedByBackend):
            be.layerNorm(data(be, 16), None, None, 4, 4, dtype)
        with pytest.raises(B.NotImplementedByBackend):
            be.groupedMatmul(1, data(be, 2, 8), data(be, 16), data(be, 16), False, 4, 4, 4, dtype)


def test_norm_and_groups_check_sizes(be):
    stat = lambda n: data(be, n, 4)  # noqa: E731
    with pytest.raises(ValueError, match="weight is smaller"):
        be.layerNorm(data(be, 16), stat(3), None, 4, 4, np.float16, out=data(be, 16))
    with pytest.raises(ValueError, match="mean is smaller"):
        be.layerNorm(data(be, 16), None, None, 4, 4, np.float16, out=data(be, 16), mean=stat(3))
    with pytest.raises(ValueError, match="rstd is smaller"):
        be.layerNormGrad(data(be, 16), data(be, 16), None, stat(4), stat(3), 4, 4, np.float16, out=data(be, 16))
    with pytest.raises(ValueError, match="offsets is smaller"):
        be.groupedMatmul(3, data(be, 3, 8), data(be, 16), data(be, 48), False, 4, 4, 4, np.float16, out=data(be, 16))
    with pytest.raises(ValueError, match="operand b is smaller"):
        be.groupedMatmul(3, data(be, 4, 8), data(be, 16), data(be, 47), False, 4, 4, 4, np.float16, out=data(be, 16))
    with pytest.raises(ValueError, match="out is smaller"):
        be.groupedMatmulWeightGrad(3, data(be, 4, 8), data(be, 16), data(be, 16), 4, 4, 4, np.float16, out=data(be, 47))
    be.groupedMatmulWeightGrad(3, data(be, 4, 8), data(be, 16), data(be, 16), 4, 4, 4, np.float16, out=data(be, 48), mark=False)
    assert len(called(be, "hc_grouped_matmul_weight_grad")) == 1


def test_adamw_plan(be):
    at = iter(range(1 << 10, 1 << 30, 256))
    new = lambda n, size: B.CUDAData(be, next(at), n * size, owns=False)  # noqa: E731
    row = lambda **k: dict(param=new(8, 4), grad=new(8, 2), moment1=new(8, 4), moment2=new(8, 4), count=8,  # noqa: E731
                           dtype=np.float32, gradDType=np.float16, **k)
    copy = new(8, 2)
    plan = be.adamWPlan([row(), row(copy=copy)])
    t = plan._table
    assert plan.count == 2 and t[0].count == 8 and t[0].param_copy is None and t[1].param_copy == copy.ptr
    assert (t[0].param_dtype, t[0].grad_dtype) == (L.HC_F32, L.HC_F16)
    grad = new(8, 2)
    plan.setGrad(1, grad)
    assert t[1].grad == grad.ptr
    with pytest.raises(ValueError, match="smaller"):
        plan.setGrad(0, new(7, 2))
    be.adamW(plan, 3, mark=False)
    (args,) = called(be, "hc_adamw")
    assert args[2:4] == (2, 3)
    with pytest.raises(ValueError, match="unknown entries"):
        be.adamWPlan([row(momentum=None)])
    with pytest.raises(ValueError, match="dtype"):
        be.adamWPlan([{k: v for k, v in row().items() if k not in ("dtype", "gradDType")}])
    with pytest.raises(ValueError, match="copy"):
        be.adamWPlan([row(copy=new(7, 2))])


def test_adamw_plan_refuses_what_two_tensors_share(be):
    at = iter(range(1 << 10, 1 << 30, 256))
    new = lambda: B.CUDAData(be, next(at), 32, owns=False)  # noqa: E731
    row = lambda **k: dict(dict(param=new(), grad=new(), moment1=new(), moment2=new(), count=8, dtype=np.float32), **k)  # noqa: E731
    tied, grad = new(), new()
    with pytest.raises(ValueError, match="param of tensor 1 overlaps param of tensor 0"):
        be.adamWPlan([row(param=tied), row(param=tied)])
    with pytest.raises(ValueError, match="overlaps"):
        be.adamWPlan([row(), row(grad=tied), row(moment2=tied)])
    with pytest.raises(ValueError, match="overlaps"):
        be.adamWPlan([row(param=B.CUDAData(be, 1 << 9, 32, owns=False)), row(moment1=B.CUDAData(be, (1 << 9) + 28, 32, owns=False))])
    be.adamWPlan([row(grad=grad), row(grad=grad)])       # a gradient is only read
    be.adamWPlan([row(param=B.CUDAData(be, 1 << 9, 32, owns=False)), row(param=B.CUDAData(be, (1 << 9) + 32, 32, owns=False))])


def test_a_new_gradient_must_not_overlap_what_the_step_writes(be):
    at = lambda p, n: B.CUDAData(be, p, n, owns=False)  # noqa: E731
    row = lambda p: dict(param=at(p, 28), grad=at(p + 64, 28), moment1=at(p + 128, 28), moment2=at(p + 192, 28), dtype="float32", count=7)  # noqa: E731
    plan = be.adamWPlan([row(4096), row(8192)])
    for start in (4096, 4096 - 24, 4096 + 24, 8192 + 128, 8192 + 192 + 24):
        with pytest.raises(ValueError, match="overlaps"):
            plan.setGrad(0, at(start, 28))
    assert plan._table[0].grad == 4096 + 64
    for start in (4096 - 28, 4096 + 28, 8192 + 64, 1024, 1 << 20):
        plan.setGrad(0, at(start, 28))
        assert plan._table[0].grad == start


def test_buffers_of_another_device_are_refused(be):
    other = B.CUDABackend.__new__(B.CUDABackend)
    other._lib, other._ctx, other.device = Recorder(), 1, 1
    beside = B.CUDABackend.__new__(B.CUDABackend)
    beside._lib, beside._ctx, beside.device = Recorder(), 1, 0
    rest = (None, None, 2, 4, "float16")
    with pytest.raises(ValueError, match="device 1"):
        be.layerNorm(data(other, 8), *rest, out=data(be, 8), mark=False)
    with pytest.raises(ValueError, match="device 1"):
        be.layerNorm(data(be, 8), *rest, out=data(other, 8), mark=False)
    be.layerNorm(data(beside, 8), *rest, out=data(be, 8), mark=False)
    assert len(called(be, "hc_layer_norm")) == 1
    other._ctx = beside._ctx = None


def test_a_loop_keeps_no_earlier_results(be):
    import weakref
    owned = lambda n: B.CUDAData(be, 512, n * 2, owns=True)  # noqa: E731
    borrowed, weight = data(be, 8), data(be, 16)
    out = be.layerNorm(borrowed, None, None, 2, 4, "float16", out=owned(8), mark=False)
    assert out._inputs == (borrowed,)
    earlier = []
    for _ in range(3):
        earlier.append(weakref.ref(out))
        out = be.matmulEpilogue(out, False, weight, False, 2, 4, 4, "float16", residual=out, out=owned(8), mark=False)
        assert out._inputs == (weight,)
    assert all(r() is None for r in earlier)
    be.layerNorm(borrowed, None, None, 2, 4, "float16", out=borrowed, mark=False)   # in place: no cycle
    assert borrowed._inputs == ()
