"""SiLU and sigmoid gates far from zero, element by element: both are small far below, the sigmoid's slope is small on both sides, and none of them
is what a difference of 1 and the sigmoid would leave of it.  Tolerances as in test_gpu_gelu_tail.py; NaN and infinite gates give what the formulas
give."""
import numpy as np
import pytest

from util import f

pytestmark = pytest.mark.gpu
TOL = {np.float16: 5e-4, np.float32: 1e-5}


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("act", ["silu", "sigmoid"])
@pytest.mark.parametrize("rows,inner,cols", [(3, 8, 256), (100, 40, 256), (5, 1, 33)])
def test_far_from_zero(rows, inner, cols, act, dtype):
    from deep8_amd import ops
    gate, factor = np.linspace(-15, 15, cols).astype(dtype), np.full(cols, 1000, dtype)
    x, w = np.zeros((rows, inner), dtype), np.zeros((inner, 2 * cols), dtype)
    x[:, 0], w[0] = 1, np.concatenate([gate, factor])
    a = gate.astype(np.float64)
    s, rest = 1 / (1 + np.exp(-a)), 1 / (1 + np.exp(a))
    value, slope, terms = (a * s, s * (1 + a * rest), s * (1 + np.abs(a) * rest)) if act == "silu" else (s, s * rest, s * rest)
    h, pre = ops.matmul_gated(x, w, act)
    assert (np.abs(f(h).astype(np.float64) - 1000 * value) <= TOL[dtype] * np.abs(1000 * value)).all()
    dh = np.zeros((rows, cols), dtype)
    dh[0] = 4
    _, dw = ops.matmul_gated_grad(x, w, pre, dh, act)
    near = 2.0 ** -25 if dtype == np.float16 else 0  # (a subnormal half's rounding)
    assert (np.abs(f(dw[0, cols:]).astype(np.float64) - 4 * value) <= TOL[dtype] * np.abs(4 * value) + near).all()
    assert (np.abs(f(dw[0, :cols]).astype(np.float64) - 4000 * slope) <= TOL[dtype] * 4000 * terms + near).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
def test_infinite_gates(act, dtype):
    from deep8_amd import ops
    gate = np.array([np.inf, np.nan, 5.0, -5.0], dtype)
    x, w, dh = np.ones((2, 1), dtype), np.concatenate([gate, np.ones(4, dtype)])[None], np.ones((2, 4), dtype)
    h, pre = ops.matmul_gated(x, w, act)
    h = f(h)
    assert (h[:, 0] == (1 if act == "sigmoid" else np.inf)).all() and (np.isnan(h[:, 1]).all() or act == "relu")
    assert np.isfinite(h[:, 2:]).all()
    _, dw = ops.matmul_gated_grad(x, w, pre, dh, act)
    assert np.isfinite(f(dw[0, 2:4])).all() and (f(dw[0, 4]) == 2 * h[0, 0]).all()
