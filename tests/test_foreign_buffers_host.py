"""Buffers that belong to another backend: results are refused, whose completion and release their owner would order on its own stream."""
import numpy as np
import pytest

from honeycrisp_b200 import _lib as L
from honeycrisp_b200 import backend as B


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return L.HC_OK
        return call


def backend(device=0):
    b = B.CUDABackend.__new__(B.CUDABackend)
    b._lib, b._ctx, b.device = Recorder(), 1, device
    return b


@pytest.fixture
def be():
    b = backend()
    yield b
    b._ctx = None


@pytest.fixture
def beside():
    b = backend()
    yield b
    b._ctx = None


AT = iter(range(1 << 12, 1 << 30, 1 << 12))


def data(be, elements, size=2):
    return B.CUDAData(be, next(AT), elements * size, owns=False)


# every result buffer of every call: (call with `r(name)` for the result named, their names)
CALLS = {
    "matmulEpilogue": (lambda be, r: be.matmulEpilogue(data(be, 12), False, data(be, 20), False, 3, 4, 5, "float16", pre=r("pre", 15), out=r("out", 15)), ("pre", "out")),
    "activationGrad": (lambda be, r: be.activationGrad(data(be, 16), data(be, 16), 4, 4, "float16", "gelu", out=r("out", 16), biasGrad=r("biasGrad", 4, 4)),
                       ("out", "biasGrad")),
    "layerNorm": (lambda be, r: be.layerNorm(data(be, 16), None, None, 4, 4, "float16", out=r("out", 16), mean=r("mean", 4, 4), rstd=r("rstd", 4, 4)),
                  ("out", "mean", "rstd")),
    "layerNormGrad": (lambda be, r: be.layerNormGrad(data(be, 16), data(be, 16), None, data(be, 4, 4), data(be, 4, 4), 4, 4, "float16", out=r("out", 16),
                                                     weightGrad=r("weightGrad", 4, 4), biasGrad=r("biasGrad", 4, 4)), ("out", "weightGrad", "biasGrad")),
    "groupedMatmul": (lambda be, r: be.groupedMatmul(1, data(be, 2, 8), data(be, 16), data(be, 16), False, 4, 4, 4, "float16", out=r("out", 16)), ("out",)),
    "groupedMatmulWeightGrad": (lambda be, r: be.groupedMatmulWeightGrad(1, data(be, 2, 8), data(be, 16), data(be, 16), 4, 4, 4, "float16", out=r("out", 16)), ("out",)),
}


@pytest.mark.parametrize("name,result", [(n, r) for n, (_, results) in CALLS.items() for r in results])
def test_a_result_of_another_backend_is_refused(be, beside, name, result):
    call, _ = CALLS[name]
    call(be, lambda n, count, size=2: data(be, count, size))
    issued = len(be._lib.calls)
    with pytest.raises(ValueError, match=f"{result} belongs to another backend"):
        call(be, lambda n, count, size=2: data(beside if n == result else be, count, size))
    assert not [n for n, _ in be._lib.calls[issued:] if n != "hc_event_destroy"] and not beside._lib.calls


def row(be, **other):
    d = dict(param=data(be, 8, 4), grad=data(be, 8, 4), moment1=data(be, 8, 4), moment2=data(be, 8, 4), copy=data(be, 8, 2), count=8, dtype=np.float32)
    return dict(d, **other)


@pytest.mark.parametrize("field", ["param", "moment1", "moment2", "copy"])
def test_a_plan_refuses_what_it_would_update_of_another_backend(be, beside, field):
    with pytest.raises(ValueError, match="belongs to another backend"):
        be.adamWPlan([row(be), row(be, **{field: data(beside, 8, 4)})])
    be.adamWPlan([row(be, grad=data(beside, 8, 4))])   # read only


def test_a_plan_of_another_backend_is_refused(be, beside):
    plan = beside.adamWPlan([row(beside)])
    with pytest.raises(ValueError, match="another backend"):
        be.adamW(plan, 1)
    assert not [n for n, _ in be._lib.calls if n == "hc_adamw"]
    beside.adamW(plan, 1)
    assert len([n for n, _ in beside._lib.calls if n == "hc_adamw"]) == 1


def test_a_plan_of_another_device_is_refused(be):
    far = backend(1)
    plan = far.adamWPlan([])
    with pytest.raises(ValueError, match="device 1"):
        be.adamW(plan, 1)
    far._ctx = None
