"""GELU of negative gates, element by element: a (1 + erf(a / sqrt 2)) / 2 is small there, and a difference of 1 and erf would leave few of its
bits.  The gate is one exact product, so what goes in is the activation and its product with the factor in fp32, and the result's
rounding.  Float16: 2^-11 = 4.9e-4 for the rounding, 1e-5 for the rest (the exponent of up to 20 in fp32 steps of 2^-20); the gradient of the
factor is rounded to half once.  Float32: the argument's and the exponential's roundings, 40 times 2^-24 at a = -5.5: 1e-5."""
import numpy as np
import pytest

import layer_oracle as lo
from util import f

pytestmark = pytest.mark.gpu
TOL = {np.float16: 5e-4, np.float32: 1e-5}


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,inner,cols", [(3, 8, 256), (100, 40, 256), (256, 64, 24576), (5, 1, 33)])  # few rows, tiles, large tiles, odd rows
def test_negative_gates(rows, inner, cols, dtype):
    from deep8_amd import ops
    gate, factor = np.linspace(-5.5, 5.5, cols).astype(dtype), np.full(cols, 1000, dtype)
    x, w = np.zeros((rows, inner), dtype), np.zeros((inner, 2 * cols), dtype)
    x[:, 0], w[0] = 1, np.concatenate([gate, factor])
    a = gate.astype(np.float64)
    value, slope = lo.gate(a, "gelu")
    tail = np.array([0.5 * lo.math.erfc(-v / 2 ** 0.5) for v in a])  # the integral itself, without the oracle's own cancellation
    value, slope = a * tail, slope - (value / np.where(a == 0, 1, a)) * (a != 0) + tail * (a != 0)
    h, pre = ops.matmul_gated(x, w, "gelu")
    assert (np.abs(f(h).astype(np.float64) - 1000 * value) <= TOL[dtype] * np.abs(1000 * value)).all()
    dh = np.zeros((rows, cols), dtype)
    dh[0] = 8
    _, dw = ops.matmul_gated_grad(x, w, pre, dh, "gelu")
    assert (np.abs(f(dw[0, cols:]).astype(np.float64) - 8 * value) <= TOL[dtype] * np.abs(8 * value) + (2.0 ** -25 if dtype == np.float16 else 0)).all()
    # the slope is a difference for gates near -0.75: against the size of its terms
    terms = tail + np.abs(a) * np.exp(-0.5 * a * a) * (2 * np.pi) ** -0.5
    assert (np.abs(f(dw[0, :cols]).astype(np.float64) - 8000 * slope) <= TOL[dtype] * 8000 * terms).all()
