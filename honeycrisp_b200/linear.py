"""`Linear` on the CUDA backend: forward and backward pass without leaving the device.

Mirrors Sources/Honeycrisp/Trainable.swift:508-547: weight `[inCount, outCount]` initialised
uniformly in +-sqrt(3)/sqrt(inCount) (`(rand - 0.5) * (sqrt(3) / 0.5 / sqrt(inCount))`), bias
`[outCount]` of zeros, forward `x . W + b` with inputs of rank > 2 flattened to
`[prod(leading dims), inCount]`.  The backward pass issues what the reference's autodiff issues
for that forward (Linalg.swift:73-80 and Tensor.swift:845-871):

    dX = matmul(a: dY, transA: false, b: W, transB: true,  transOut: false)
    dW = matmul(a: X,  transA: true,  b: dY, transB: false, transOut: false)
    db = sum of dY over its rows            (reduceBroadcast of the broadcast add)

Parameter dtypes follow the reference exactly (Trainable.swift:514-544): the weight is created
in `dtype`, the bias ALWAYS in float32 (`Tensor(zeros: [outCount])`), and the forward pass uses
`weight.cast(castParams ?? weight.dtype)` and `bias.cast(castParams ?? bias.dtype)`.  So a layer
computing in float16 is either `Linear(dtype: .float16, castParams: .float16)` (float16 weight,
float32 bias cast on use) or `Linear(dtype: .float32, castParams: .float16)` (float32 master
weights cast on every call); a float16 layer with a bias and no castParams adds float16 to
float32, which the reference's binary ops refuse, and so does this class.  Gradients arrive in the
compute dtype and are cast back to each parameter's dtype (the backward of `cast`).

With an activation or a residual the layer runs as one product with a fused epilogue instead,

    pre = x . W + b,   out = activation(pre) + residual          (float32 throughout, rounded once)

and its backward pass starts with the gradient through the activation, which brings the bias gradient along.  A layer in front of
it can take its own activation's slope into this layer's input gradient (`inputPre`, `inputActivation`): the product
dX = dPre . W^T then leaves as the gradient of that layer's pre-activation.

Weights come from numpy's generator, not from Honeycrisp's Philox stream, so parameter values
differ from a Honeycrisp `Linear` with the same seed; shapes, ranges and arithmetic do not.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import numpy as np

from .backend import CUDABackend, CUDAData, DType, _as_dtype


class Linear:
    def __init__(self, backend: CUDABackend, inCount: int, outCount: int, dtype=np.float32, castParams=None,
                 bias: bool = True, seed: int = 0, activation: Optional[str] = None):
        self.backend, self.inCount, self.outCount = backend, int(inCount), int(outCount)
        self.dtype = _as_dtype(dtype)                                    # of the weight
        self.castParams = _as_dtype(castParams) if castParams is not None else None
        self.biasDType = DType.float32                                   # Trainable.swift:524
        self.activation = activation if activation != "none" else None
        rng = np.random.default_rng(seed)
        w = (rng.random((inCount, outCount), dtype=np.float32) - 0.5) * (math.sqrt(3.0) / 0.5 / math.sqrt(inCount))
        self.weight = backend.collection(w.astype(self.dtype.numpy), self.dtype)
        self.bias = backend.collection(np.zeros(outCount, dtype=np.float32), DType.float32) if bias else None
        self.weightGrad: Optional[CUDAData] = None
        self.biasGrad: Optional[CUDAData] = None

    @property
    def computeDType(self) -> DType:
        return self.castParams or self.dtype

    def _castWeight(self) -> CUDAData:
        ct = self.computeDType
        if ct == self.dtype:
            return self.weight
        return self.backend.cast(self.weight, self.inCount * self.outCount, self.dtype, ct)

    def _castBias(self) -> Optional[CUDAData]:
        if self.bias is None:
            return None
        bt = self.castParams or self.biasDType
        if bt != self.computeDType:
            # h is in the weight's dtype, the bias in float32: the reference's `h + bias` asserts
            raise ValueError(f"Linear: bias is {bt.value} but the product is {self.computeDType.value}; "
                             f"pass castParams (Trainable.swift:540-544)")
        if bt == self.biasDType:
            return self.bias
        return self.backend.cast(self.bias, self.outCount, self.biasDType, bt)

    def __call__(self, x, shape: Sequence[int], residual=None) -> Tuple[CUDAData, list]:
        """Forward.  `x` holds a dense tensor of `shape`, in the layer's compute dtype, whose last
        dimension is inCount; returns the output buffer and its shape.  `residual`, of the output's shape, is added behind
        the activation."""
        if self.activation is None and residual is None:
            shape, rows = self._rows(shape)
            out = self.backend.linearForward(x, self._castWeight(), self._castBias(), rows, self.inCount, self.outCount,
                                             self.computeDType)
            return out, shape[:-1] + [self.outCount]
        return self._fused(x, shape, residual, None)

    def forwardKeepingPre(self, x, shape: Sequence[int], residual=None) -> Tuple[CUDAData, list, CUDAData]:
        """Forward for training a layer with an activation: also returns the activation's input, for `backward`."""
        _, rows = self._rows(shape)
        pre = self.backend.allocate(rows * self.outCount * self.computeDType.byteSize)
        out, outShape = self._fused(x, shape, residual, pre)
        return out, outShape, pre

    def _rows(self, shape):
        shape = list(int(s) for s in shape)
        assert shape and shape[-1] == self.inCount, f"last dimension must be {self.inCount}: {shape}"
        return shape, int(np.prod(shape[:-1])) if len(shape) > 1 else 1

    def _fused(self, x, shape, residual, pre):
        shape, rows = self._rows(shape)
        out = self.backend.matmulEpilogue(x, False, self._castWeight(), False, rows, self.inCount, self.outCount, self.computeDType,
                                          activation=self.activation, bias=self._castBias(), residual=residual, pre=pre)
        return out, shape[:-1] + [self.outCount]

    def backward(self, x, shape: Sequence[int], outGrad, pre=None, inputPre=None, inputActivation: Optional[str] = None) -> CUDAData:
        """Backward for the forward call on (`x`, `shape`): returns dX and accumulates the
        parameter gradients (Param.addGrad, Trainable.swift:258-266).  `pre` is what forwardKeepingPre returned, for a layer with
        an activation (a residual's gradient is outGrad itself).  With `inputPre` and `inputActivation`, the input of this
        layer is inputActivation(inputPre) and what comes back is the gradient of inputPre."""
        shape = list(int(s) for s in shape)
        rows = int(np.prod(shape[:-1])) if len(shape) > 1 else 1
        be = self.backend
        ct = self.computeDType
        db = None
        if self.activation is not None:
            if pre is None:
                raise ValueError("Linear: the backward pass of a layer with an activation needs `pre` (forwardKeepingPre)")
            outGrad, db = be.activationGrad(outGrad, pre, rows, self.outCount, ct, self.activation, biasGrad=self.bias is not None)
        return self._backwardOfPre(x, rows, outGrad, db, inputPre, inputActivation)

    def backwardOfPre(self, x, shape: Sequence[int], preGrad) -> CUDAData:
        """Backward from the gradient of the activation's input, as the layer behind returns it (`inputPre`)."""
        _, rows = self._rows(shape)
        return self._backwardOfPre(x, rows, preGrad, None, None, None)

    def _backwardOfPre(self, x, rows: int, outGrad, db, inputPre, inputActivation) -> CUDAData:
        be = self.backend
        ct = self.computeDType
        if inputPre is not None:
            dx = be.matmulEpilogue(outGrad, False, self._castWeight(), True, rows, self.outCount, self.inCount, ct,
                                   activation=inputActivation, gradPre=inputPre)
        else:
            dx = be.matmul(outGrad, False, self._castWeight(), True, False, rows, self.outCount, self.inCount, ct)
        dw = be.matmul(x, True, outGrad, False, False, self.inCount, rows, self.outCount, ct)
        if ct != self.dtype:                          # backward of weight.cast(castParams)
            dw = be.cast(dw, self.inCount * self.outCount, ct, self.dtype)
        self.weightGrad = dw if self.weightGrad is None else be.add(self.weightGrad, dw, self.inCount * self.outCount,
                                                                    self.dtype)
        if self.bias is not None:
            if db is None:
                db = be.columnSum(outGrad, rows, self.outCount, ct)
                if ct != self.biasDType:              # backward of bias.cast(castParams)
                    db = be.cast(db, self.outCount, ct, self.biasDType)
            self.biasGrad = db if self.biasGrad is None else be.add(self.biasGrad, db, self.outCount, self.biasDType)
        return dx

    def parameters(self):
        """(buffer, gradient, element count, dtype) of each parameter, for AdamW."""
        out = [(self.weight, self.weightGrad, self.inCount * self.outCount, self.dtype)]
        if self.bias is not None:
            out.append((self.bias, self.biasGrad, self.outCount, self.biasDType))
        return out

    def zeroGrad(self) -> None:
        self.weightGrad = self.biasGrad = None
