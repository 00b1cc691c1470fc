"""What stands around `Linear` in a feed-forward block: LayerNorm, the block itself, its form by experts, and AdamW.

Each class holds device buffers and issues the backend's calls, in the manner of `Linear`: forward returns what the backward pass
needs, backward returns the input's gradient and accumulates the parameters'.  LayerNorm follows Trainable.swift's
LayerNorm (float32 gain of ones and bias of zeros, epsilon 1e-5), AdamW its Optimizer.swift's Adam with decoupled decay.
"""
from __future__ import annotations

from typing import Optional, Sequence

import numpy as np

from .backend import AdamWPlan, CUDABackend, CUDAData, DType, _as_dtype
from .linear import Linear


def _accumulate(be: CUDABackend, old: Optional[CUDAData], new: CUDAData, count: int, dtype: DType) -> CUDAData:
    return new if old is None else be.add(old, new, count, dtype)


class LayerNorm:
    """Normalisation over the last dimension, with float32 parameters whatever the input's dtype."""

    def __init__(self, backend: CUDABackend, width: int, dtype=np.float32, epsilon: float = 1e-5):
        self.backend, self.width, self.dtype, self.epsilon = backend, int(width), _as_dtype(dtype), float(epsilon)
        self.weight = backend.constant(1.0, width, DType.float32)
        self.bias = backend.constant(0.0, width, DType.float32)
        self.weightGrad: Optional[CUDAData] = None
        self.biasGrad: Optional[CUDAData] = None

    def __call__(self, x, rows: int):
        """(output, statistics): the second is what backward needs."""
        be = self.backend
        mean, rstd = be.allocate(rows * 4), be.allocate(rows * 4)
        out = be.layerNorm(x, self.weight, self.bias, rows, self.width, self.dtype, epsilon=self.epsilon, mean=mean, rstd=rstd)
        return out, (mean, rstd)

    def backward(self, x, rows: int, outGrad, statistics) -> CUDAData:
        be = self.backend
        dx, dw, db = be.layerNormGrad(outGrad, x, self.weight, statistics[0], statistics[1], rows, self.width, self.dtype)
        self.weightGrad = _accumulate(be, self.weightGrad, dw, self.width, DType.float32)
        self.biasGrad = _accumulate(be, self.biasGrad, db, self.width, DType.float32)
        return dx

    def parameters(self):
        return [(self.weight, self.weightGrad, self.width, DType.float32), (self.bias, self.biasGrad, self.width, DType.float32)]

    def zeroGrad(self) -> None:
        self.weightGrad = self.biasGrad = None


class FeedForward:
    """out = x + down(activation(up(norm(x)))): two fused products forward, and backward one that carries the gradient through
    the activation between the weight gradients."""

    def __init__(self, backend: CUDABackend, width: int, hidden: int, activation: str = "gelu", dtype=np.float32, castParams=None,
                 seed: int = 0):
        self.backend, self.width, self.hidden, self.activation = backend, int(width), int(hidden), activation
        self.up = Linear(backend, width, hidden, dtype, castParams, seed=seed, activation=activation)
        self.down = Linear(backend, hidden, width, dtype, castParams, seed=seed + 1)
        self.dtype = self.up.computeDType
        self.norm = LayerNorm(backend, width, self.dtype)

    def __call__(self, x, rows: int):
        """(output, saved): the second is what backward needs."""
        n, statistics = self.norm(x, rows)
        h, _, pre = self.up.forwardKeepingPre(n, [rows, self.width])
        out, _ = self.down(h, [rows, self.hidden], residual=x)
        return out, (x, rows, n, statistics, h, pre)

    def backward(self, outGrad, saved) -> CUDAData:
        be = self.backend
        x, rows, n, statistics, h, pre = saved
        dPre = self.down.backward(h, [rows, self.hidden], outGrad, inputPre=pre, inputActivation=self.activation)
        dn = self.up.backwardOfPre(n, [rows, self.width], dPre)
        dx = self.norm.backward(x, rows, dn, statistics)
        return be.add(outGrad, dx, rows * self.width, self.dtype)   # the residual's share

    def parameters(self):
        return self.norm.parameters() + self.up.parameters() + self.down.parameters()

    def zeroGrad(self) -> None:
        for m in (self.norm, self.up, self.down):
            m.zeroGrad()


class Experts:
    """One weight matrix [inCount, outCount] for each of `groups` experts, applied to rows that are sorted by expert: rows
    offsets[g] to offsets[g + 1] meet matrix g.  The offsets (int64, groups + 1) stay on the device."""

    def __init__(self, backend: CUDABackend, groups: int, inCount: int, outCount: int, dtype=np.float32, seed: int = 0):
        self.backend, self.groups, self.inCount, self.outCount = backend, int(groups), int(inCount), int(outCount)
        self.dtype = _as_dtype(dtype)
        rng = np.random.default_rng(seed)
        w = (rng.random((groups, inCount, outCount), dtype=np.float32) * 2 - 1) * np.float32(np.sqrt(3.0 / inCount))
        self.weight = backend.collection(w.astype(self.dtype.numpy), self.dtype)
        self.weightGrad: Optional[CUDAData] = None

    def __call__(self, x, offsets, rows: int) -> CUDAData:
        out = self.backend.constant(0.0, rows * self.outCount, self.dtype)   # rows of no expert
        return self.backend.groupedMatmul(self.groups, offsets, x, self.weight, False, rows, self.inCount, self.outCount, self.dtype, out=out)

    def backward(self, x, offsets, rows: int, outGrad) -> CUDAData:
        be = self.backend
        dx = be.constant(0.0, rows * self.inCount, self.dtype)
        be.groupedMatmul(self.groups, offsets, outGrad, self.weight, True, rows, self.outCount, self.inCount, self.dtype, out=dx)
        dw = be.groupedMatmulWeightGrad(self.groups, offsets, x, outGrad, rows, self.inCount, self.outCount, self.dtype)
        self.weightGrad = _accumulate(be, self.weightGrad, dw, self.groups * self.inCount * self.outCount, self.dtype)
        return dx

    def parameters(self):
        return [(self.weight, self.weightGrad, self.groups * self.inCount * self.outCount, self.dtype)]

    def zeroGrad(self) -> None:
        self.weightGrad = None


class AdamW:
    """AdamW over the parameters of modules such as the above, one launch a step.  A module may replace a parameter's buffer between
    steps (`layer.weight = ...`): the new one is trained from then on, with the moments that stood in its place.  Number and lengths of the
    parameters are the first step's."""

    def __init__(self, backend: CUDABackend, modules: Sequence, learningRate: float = 1e-3, beta1: float = 0.9, beta2: float = 0.999,
                 epsilon: float = 1e-8, weightDecay: float = 0.01):
        self.backend, self.modules = backend, list(modules)
        self.hyper = dict(learningRate=learningRate, beta1=beta1, beta2=beta2, epsilon=epsilon, weightDecay=weightDecay)
        self.stepCount = 0
        self.plan: Optional[AdamWPlan] = None
        self.moments = []
        self._planned = []   # the plan's parameters: (buffer, elements)

    def step(self) -> None:
        """Updates every parameter from its accumulated gradient; every parameter needs one."""
        be = self.backend
        parameters = [p for m in self.modules for p in m.parameters()]
        if any(g is None for _, g, _, _ in parameters):
            raise ValueError("AdamW: a parameter has no gradient")
        if self.plan is None:
            self.moments = [(be.constant(0.0, n, DType.float32), be.constant(0.0, n, DType.float32)) for _, _, n, _ in parameters]
        elif len(parameters) != len(self._planned):
            raise ValueError(f"AdamW: {len(parameters)} parameters, {len(self._planned)} at the first step")
        else:
            for i, ((_, _, n, _), (_, before)) in enumerate(zip(parameters, self._planned)):
                if n != before:
                    raise ValueError(f"AdamW: parameter {i} has {n} elements, {before} at the first step")
        if self.plan is None or any(p is not q for (p, _, _, _), (q, _) in zip(parameters, self._planned)):
            self.plan = be.adamWPlan([dict(param=p, grad=g, moment1=m, moment2=v, count=n, dtype=t)
                                      for (p, g, n, t), (m, v) in zip(parameters, self.moments)])
            self._planned = [(p, n) for p, _, n, _ in parameters]
        else:
            for i, (_, g, _, _) in enumerate(parameters):
                self.plan.setGrad(i, g)
        be.adamW(self.plan, self.stepCount + 1, **self.hyper)
        self.stepCount += 1

    def zeroGrad(self) -> None:
        for m in self.modules:
            m.zeroGrad()
