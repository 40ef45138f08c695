"""d8_layer_norm over its input, and d8_layer_norm_grad over either of its: rows that would lie elsewhere than those they are made from are refused (one would be
written where another has still to be read), before anything is launched: the tensors need not be there, nor a device."""
import pytest

from deep8_amd import capi

P, Q = 64, 1 << 20


@pytest.mark.parametrize("rows,code", [(4, 10001), (2, 10001), (0, 0)])
def test_forward(rows, code):
    lib = capi.load()
    assert lib.d8_layer_norm(capi.FLOAT32, P, 8, None, None, P, 16, rows, 8, 1e-5, None) == code
    assert lib.d8_layer_norm(capi.FLOAT32, P, 16, None, None, P, 8, rows, 8, 1e-5, None) == code


@pytest.mark.parametrize("over", ["x", "dy"])
@pytest.mark.parametrize("rows,code", [(4, 10001), (2, 10001), (0, 0)])
def test_gradient(over, rows, code):
    lib = capi.load()
    dx = P if over == "x" else Q
    assert lib.d8_layer_norm_grad(capi.FLOAT16, P, 8, None, Q, 8, dx, 16, None, None, rows, 8, 1e-5, 3, None, 0, None) == code
    assert lib.d8_layer_norm_grad(capi.FLOAT16, P, 16, None, Q, 16, dx, 8, None, None, rows, 8, 1e-5, 1, None, 0, None) == code
