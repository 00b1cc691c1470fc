"""The optimiser over modules, on a library that only writes its calls down: which buffers a step hands over."""
import numpy as np
import pytest

from honeycrisp_b200 import AdamW
from honeycrisp_b200 import _lib as L
from honeycrisp_b200 import backend as B


class Recorder:
    """A library whose calls succeed and are written down; each allocation has an address of its own."""

    def __init__(self):
        self.calls, self.next = [], 1 << 20

    def __getattr__(self, name):
        def call(*args):
            if name == "hc_alloc":
                args[2]._obj.value, self.next = self.next, self.next + (args[1] + 255) // 256 * 256
            # a table is the plan's own memory: what it holds now
            self.calls.append((name, args, [(t.param, t.grad, t.moment1, t.moment2, t.count) for t in args[1][: args[2]]] if name == "hc_adamw" else None))
            return L.HC_OK
        return call


@pytest.fixture
def be():
    b = B.CUDABackend.__new__(B.CUDABackend)
    b._lib, b._ctx, b.device = Recorder(), 1, 0
    yield b
    b._ctx = None


class Module:
    def __init__(self, be, *counts):
        self.be, self.counts = be, counts
        self.weights = [be.allocate(n * 4) for n in counts]
        self.newGrads()

    def newGrads(self):
        self.grads = [self.be.allocate(n * 4) for n in self.counts]

    def parameters(self):
        return [(w, g, n, B.DType.float32) for w, g, n in zip(self.weights, self.grads, self.counts)]


def steps(be):
    return [t for name, _, t in be._lib.calls if name == "hc_adamw"]


def test_a_replaced_parameter_is_the_one_that_is_trained(be):
    m = Module(be, 40, 7)
    optimiser = AdamW(be, [m])
    optimiser.step()
    old, m.weights[1] = m.weights[1], be.allocate(28)
    m.newGrads()
    optimiser.step()
    first, second = steps(be)
    assert [t[0] for t in first] == [m.weights[0].ptr, old.ptr]
    assert [t[0] for t in second] == [w.ptr for w in m.weights] and [t[1] for t in second] == [g.ptr for g in m.grads]
    assert [t[2:] for t in second] == [t[2:] for t in first]      # its moments go on
    m.newGrads()
    optimiser.step()
    assert [t[:2] for t in steps(be)[2]] == [(w.ptr, g.ptr) for w, g in zip(m.weights, m.grads)]


def test_other_parameters_than_the_first_steps_are_refused(be):
    m, other = Module(be, 40, 7), Module(be, 5)
    optimiser = AdamW(be, [m, other])
    optimiser.step()
    optimiser.modules = [m]
    with pytest.raises(ValueError, match="parameters"):
        optimiser.step()
    optimiser.modules = [m, other]
    other.counts, other.weights = (6,), [be.allocate(24)]
    other.newGrads()
    with pytest.raises(ValueError, match="elements"):
        optimiser.step()
    assert len(steps(be)) == 1


def test_a_step_that_failed_does_not_count(be):
    m = Module(be, 40)
    optimiser = AdamW(be, [m])
    optimiser.step()
    optimiser.hyper["epsilon"], good = -1.0, optimiser.hyper["epsilon"]
    refuse = lambda *a: L.HC_ERR_INVALID_ARGUMENT if a[7] < 0 else L.HC_OK  # noqa: E731
    be._lib.hc_adamw, be._lib.hc_last_error = refuse, lambda *a: b"epsilon must not be negative"
    with pytest.raises(ValueError, match="epsilon"):
        optimiser.step()
    optimiser.hyper["epsilon"] = good
    del be._lib.hc_adamw
    optimiser.step()
    assert [args[3] for name, args, _ in be._lib.calls if name == "hc_adamw"] == [1, 2] and optimiser.stepCount == 2
