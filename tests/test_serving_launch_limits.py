"""Sizes whose launches would have more threads than there can be are refused before anything is launched (the tensors need not be there, nor a device): a call
that failed at its second launch would have changed a part of its results."""
import pytest

from deep8_amd import capi

P, MANY = 64, 1 << 60


@pytest.mark.parametrize("cols,code", [((1 << 27) + 1, 10001), (1 << 29, 10001)])
def test_norm_gradients_sums(cols, code):
    lib = capi.load()
    for dw, db in ((P, P), (P, None), (None, P)):
        assert lib.d8_layer_norm_grad(capi.FLOAT16, P, cols, None, P, cols, P, cols, dw, db, 1, cols, 1e-5, 3, P, MANY, None) == code
        assert lib.d8_layer_norm_grad(capi.FLOAT16, P, cols, None, P, cols, None, 0, dw, db, 0, cols, 1e-5, 3, P, MANY, None) == code
    assert lib.d8_layer_norm_grad_scratch_bytes(capi.FLOAT16, 1, cols) == 0


@pytest.mark.parametrize("cols", [(1 << 29) + 1, (1 << 31) - 1])
def test_columns(cols):
    lib = capi.load()
    assert lib.d8_quantize_columns(capi.FLOAT16, P, cols, 1, cols, P, P, None) == 10001
