"""How near the float32 activations and their slopes come to the functions, over a dense sweep of z from -13 to 13, on every path that computes them.

The room follows the arithmetic, operation by operation, with u = 2^-24 for a rounded one and 4u for expf (two steps, CUDA's stated bound):

  GELU  The normal distribution's tail is t R(t) e^(-y^2/2), t = 1 / (1 + 0.3 y), y = |z|, R of degree 7.  The fit is off by 1.66e-7 at most
        (the coefficients as float32, evaluated in float64 over y <= 14).  Its evaluation adds at most 8.4 u: the roundings of the eight
        steps weighted by what follows each (3.1 u at y = 0) and t's two, weighted by the sensitivity of t R(t) (up to 2.7).  Two
        products and the exponential add 6 u, the exponent's own rounding y^2/2 u.
  SiLU, tanh GELU   z / (1 + e^-a), a the exponent (exact for SiLU): e^-a is off by 4 u and a's error, of which 1 / (1 + e^-a) takes
        the share e^-a / (1 + e^-a), and the sum, the quotient and the product add u each.  Where e^-a leaves float32's range (a < -88.7) the
        result is zero for values below |z| 2^-128.

The same sums are made for the slopes S + z S' below.  float16's exponential on float32 results, at three times the exponent's error and
more, does not fit in this room for |z| near 13.
"""
import numpy as np
import pytest

import operator_reference as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["relu", "gelu", "gelu_tanh", "silu"]
C1 = 2 * np.sqrt(2 / np.pi)      # the tanh form's exponent is C1 z + C3 z^3
C3 = C1 * 0.044715


@pytest.fixture(scope="module")
def be():
    from honeycrisp_b200 import CUDABackend
    b = CUDABackend(0)
    yield b
    b.checkDeviceStatus()
    b.close()


def tail_room(z):
    return 1.66e-7 + (8.4 + 6 + z * z / 2) * U


def exponent(z, name):
    """a of 1 / (1 + e^-a), and its absolute error: constants of one and four roundings, two products, two sums."""
    if name == "silu":
        return z, 0 * z
    a = C1 * z + C3 * z ** 3
    return a, (np.abs(C1 * z) + 4 * np.abs(C3 * z ** 3) + 2 * np.abs(a)) * U


def value_room(z, name):
    """Absolute room of activation(z)."""
    y = np.abs(ref.activation(z, name))
    if name == "relu":
        return 0 * z
    if name == "gelu":
        tail = ref.phi(-np.abs(z))
        return np.abs(z) * tail * tail_room(z) + 2 * U * y
    a, da = exponent(z, name)
    share = 1 - ref.sigmoid(a)
    return y * ((da + 4 * U) * share + 3 * U) + np.abs(z) * 2.0 ** -127


def slope_room(z, name):
    s = np.abs(ref.slope(z, name))
    if name == "relu":
        return 0 * z
    if name == "gelu":
        tail, peak = ref.phi(-np.abs(z)), np.abs(z) * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
        return tail * tail_room(z) + U * ref.phi(z) + peak * (2 + 4 + z * z / 2) * U + 2 * U * s
    a, da = exponent(np.abs(z), name)
    sigma = ref.sigmoid(exponent(z, name)[0])
    inner = np.abs(z) * (C1 + 3 * C3 * z * z) if name == "gelu_tanh" else np.abs(z)
    second = inner * ref.sigmoid(a) * ref.sigmoid(-a)
    return sigma * (da + 7 * U) + second * (7 * U + da + 4 * U + 6 * U) + 2 * U * s + inner * 2.0 ** -126


@pytest.mark.parametrize("name", ACTS)
def test_slopes(be, name):
    z = np.linspace(-13, 13, 400001).astype(np.float32)
    one = np.ones_like(z)
    z64 = z.astype(np.float64)
    for cols in (1, 4):          # single elements, and 16-byte pieces
        n = z.size // 4 * 4
        got, _ = be.activationGrad(one[:n], z[:n], n // cols, cols, np.float32, name, biasGrad=False)
        ref.within(got.onCPU(np.float32)[:n], ref.slope(z64[:n], name), 1.01 * slope_room(z64[:n], name), np.float32)


def grid():
    """z[i, j] = coarse[i] + fine[j], exactly, as a product of two terms: multiples of 1/4 from -13 on, and of 2^-12 below 1/4."""
    return (np.arange(-52, 52) / 4).astype(np.float32), (np.arange(1024) / 4096).astype(np.float32)


def operands(coarse, fine, inner):
    a, b = np.zeros((coarse.size, inner), np.float32), np.zeros((inner, fine.size), np.float32)
    a[:, 0], b[0], a[:, inner - 1], b[inner - 1] = coarse, 1, 1, fine
    return a, b


# (rows at a time, contracted length, kernel): CUDA cores, few rows, tensor cores, tensor cores with the contraction cut
PATHS = {"cuda_cores": (104, 2, "SIMT"), "few_rows": (8, 40, "SIMT"), "tensor": (104, 64, "TENSOR"), "cut": (104, 8192, "TENSOR")}


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("path", list(PATHS))
def test_products(be, path, name):
    from honeycrisp_b200 import _lib
    rows, inner, kernel = PATHS[path]
    coarse, fine = grid()
    for first in range(0, coarse.size, rows):
        c = coarse[first: first + rows]
        a, b = operands(c, fine, inner)
        z = c[:, None].astype(np.float64) + fine[None].astype(np.float64)
        pre = be.allocate(z.size * 4)
        out = be.matmulEpilogue(a, False, b, False, c.size, inner, fine.size, np.float32, activation=name, pre=pre)
        assert be.lastLaunchInfo()["kernel"] == getattr(_lib, f"HC_KERNEL_{kernel}")
        assert np.array_equal(pre.onCPU(np.float32)[: z.size], z.astype(np.float32).reshape(-1))
        ref.within(out.onCPU(np.float32)[: z.size], ref.activation(z, name), 1.01 * value_room(z, name), np.float32)
        # times a slope: the product is one everywhere, the pre-activations any float32
        a[:, 0], a[:, inner - 1] = 1, 0
        rng = np.random.default_rng(first)
        kept = rng.uniform(-13, 13, z.shape).astype(np.float32)
        out = be.matmulEpilogue(a, False, b, False, c.size, inner, fine.size, np.float32, activation=name, gradPre=kept)
        k64 = kept.astype(np.float64)
        ref.within(out.onCPU(np.float32)[: z.size], ref.slope(k64, name), 1.01 * slope_room(k64, name), np.float32)
