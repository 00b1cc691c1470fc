"""Plain float64 forms of the feed-forward block's operators, and the comparison the tests make.

Rounding a value to a type is off by at most half a step: 2^-11 of the value in float16 (2^-25 below its normals), 2^-24 in
float32.  A product of length K summed in float32 is off by at most K 2^-23 of the sum of magnitudes (each addition
of the tensor core truncates); float32 operands as two TF32 halves leave out 2^-20 of it and round 2^-20 more.
"""
import math

import numpy as np

HALF_STEP = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24}
SMALLEST = {np.float16: 2.0 ** -25, np.float32: 2.0 ** -126}   # half a step of float16's subnormals; float32 may flush
# Both types take the same fit, off by 1.7e-7.  float16 results take the hardware's exponential (2 + 1.2 |t| steps of 2^-23
# for e^t, |t| < 90 where the value is not yet below float16's range).  For float32 this is the exponent's rounding at its
# largest, z^2 / 2 * 2^-23 with z <= 14, wherever z lies; test_activation_accuracy_gpu.py has the room by z.
ACT_RELATIVE = {np.float16: 2.0e-5, np.float32: 1.5e-5}

_erfc = np.vectorize(math.erfc, otypes=[np.float64])


def phi(z):
    return _erfc(-z / math.sqrt(2.0)) / 2


def sigmoid(t):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-t))


_C = math.sqrt(2 / math.pi)


def activation(z, name):
    if name == "relu":
        return np.where(z < 0, 0.0, z)
    if name == "gelu":
        return z * phi(z)
    if name == "gelu_tanh":
        return z * sigmoid(2 * _C * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * sigmoid(z)
    return z


def slope(z, name):
    if name == "relu":
        return np.where(z <= 0, 0.0, 1.0)
    if name == "gelu":
        return phi(z) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        s = sigmoid(2 * _C * (z + 0.044715 * z ** 3))
        return s + z * s * (1 - s) * 2 * _C * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = sigmoid(z)
        return s + z * s * (1 - s)
    return np.ones_like(z)


def product_error(a, b, dtype):
    """Bound of each element's error of a float32-accumulated product of a[.., K] and b[K, ..]."""
    mags = np.abs(a.astype(np.float64)) @ np.abs(b.astype(np.float64))
    return mags * (a.shape[-1] * 2.0 ** -23 + (2.0 ** -19 if dtype == np.float32 else 0.0))


def within(got, want, error, dtype):
    """`error`: how far the float32 value may be before it is rounded to `dtype`; names the worst element."""
    got, want = np.asarray(got).astype(np.float64).reshape(-1), np.asarray(want, np.float64).reshape(-1)
    error = np.broadcast_to(np.asarray(error, np.float64), np.asarray(want).shape).reshape(-1) if np.ndim(error) == 0 else np.asarray(error, np.float64).reshape(-1)
    top = float(np.finfo(dtype).max)
    room = error + HALF_STEP[dtype] * (np.abs(want) + error) + SMALLEST[dtype]
    over = np.abs(want) + room >= top          # may round to infinity
    bad = ~(np.abs(got - want) <= room) & ~(over & np.isinf(got) & (np.sign(got) == np.sign(want)))
    if bad.any():
        i = int(np.argmax(np.where(bad, np.abs(got - want) / room, 0)))
        raise AssertionError(f"{int(bad.sum())} of {bad.size} outside; at {i}: {got[i]!r}, not {want[i]!r} +- {room[i]:.3g}")
