"""A buffer that has been freed is refused wherever it is passed; as an optional argument its null address would read as "none given"."""
import numpy as np
import pytest

from honeycrisp_b200 import _lib as L
from honeycrisp_b200 import backend as B


class Recorder:
    def __init__(self):
        self.calls, self.next = [], 1 << 20

    def __getattr__(self, name):
        def call(*args):
            if name == "hc_alloc":
                args[2]._obj.value, self.next = self.next, self.next + (args[1] + 255) // 256 * 256
            self.calls.append(name)
            return L.HC_OK
        return call


@pytest.fixture
def be():
    b = B.CUDABackend.__new__(B.CUDABackend)
    b._lib, b._ctx, b.device = Recorder(), 1, 0
    yield b
    b._ctx = None


def freed(be, elements, size=2):
    d = be.allocate(elements * size)
    d.free()
    return d


CASES = {
    "bias": lambda be, d: be.matmulEpilogue(d(12), False, d(20), False, 3, 4, 5, "float16", bias=freed(be, 5)),
    "residual": lambda be, d: be.matmulEpilogue(d(12), False, d(20), False, 3, 4, 5, "float16", residual=freed(be, 15)),
    "pre": lambda be, d: be.matmulEpilogue(d(12), False, d(20), False, 3, 4, 5, "float16", pre=freed(be, 15)),
    "gradPre": lambda be, d: be.matmulEpilogue(d(12), False, d(20), False, 3, 4, 5, "float16", gradPre=freed(be, 15)),
    "operand b": lambda be, d: be.matmulEpilogue(d(12), False, freed(be, 20), False, 3, 4, 5, "float16"),
    "biasGrad": lambda be, d: be.activationGrad(d(16), d(16), 4, 4, "float16", "gelu", biasGrad=freed(be, 4, 4)),
    "weight": lambda be, d: be.layerNorm(d(16), freed(be, 4, 4), None, 4, 4, "float16"),
    "mean": lambda be, d: be.layerNorm(d(16), None, None, 4, 4, "float16", mean=freed(be, 4, 4)),
    "rstd": lambda be, d: be.layerNormGrad(d(16), d(16), None, d(4, 4), freed(be, 4, 4), 4, 4, "float16"),
    "weightGrad": lambda be, d: be.layerNormGrad(d(16), d(16), None, d(4, 4), d(4, 4), 4, 4, "float16", weightGrad=freed(be, 4, 4)),
    "out": lambda be, d: be.groupedMatmul(1, d(2, 8), d(16), d(16), False, 4, 4, 4, "float16", out=freed(be, 16)),
    "param_copy": lambda be, d: be.adamWPlan([dict(param=d(8, 4), grad=d(8, 4), moment1=d(8, 4), moment2=d(8, 4), copy=freed(be, 8), count=8, dtype=np.float32)]),
}


@pytest.mark.parametrize("what", sorted(CASES))
def test_a_freed_buffer_is_refused(be, what):
    with pytest.raises(ValueError, match=f"{what} has been freed"):
        CASES[what](be, lambda n, size=2: be.allocate(n * size))
    assert not set(be._lib.calls) - {"hc_alloc", "hc_free", "hc_event_destroy"}


def test_nothing_needs_no_memory(be):
    empty = B.CUDAData(be, 0, 0, owns=False)
    be.layerNorm(empty, None, None, 0, 4, "float16", mark=False)
    assert be._lib.calls[-1] != "hc_alloc" and "hc_layer_norm" in be._lib.calls
