"""d8_matmul_gated on tensors that start anywhere, with the scratch that its query gives for them, and its gradients, whose query counts on
nothing."""
import numpy as np
import pytest

import layer_oracle as lo
from test_gpu_matmul_gated import TOL, _inputs, _near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("size", [(3, 200, 72), (4, 4096, 512), (100, 100, 100), (257, 72, 200), (256, 64, 24576)])
@pytest.mark.parametrize("off", [(1, 0), (0, 1), (3, 5)])
def test_anywhere(size, off, dtype):
    from deep8_amd import capi
    from deep8_amd.capi import DeviceArray, check
    lib, dt, es = capi.init(), capi.dtype_id(dtype), np.dtype(dtype).itemsize
    x, w, dh = _inputs(*size, dtype)
    rows, inner, cols = size

    def put(a, off):
        room = DeviceArray.from_numpy(np.concatenate([np.full(off, np.nan, dtype), a.ravel(), np.full(8, np.nan, dtype)]))
        return room, room.ptr + off * es

    (xr, xp), (wr, wp), (gr, gp) = put(x, off[0]), put(w, off[1]), put(dh, off[0])
    h, pre = DeviceArray((rows, cols), dtype), DeviceArray((rows, 2 * cols), dtype)
    nb = lib.d8_matmul_gated_scratch_bytes(dt, 2, rows, inner, cols)
    assert nb >= lib.d8_matmul_gated_scratch_bytes(dt, 0, rows, inner, cols)
    ws = DeviceArray((max(nb, 16) + 16,), np.uint8)
    ws.copy_from(np.full(ws.shape, 7, np.uint8))
    check(lib.d8_matmul_gated(dt, xp, rows, inner, wp, cols, 0, pre.ptr, h.ptr, ws.ptr, nb, None))
    capi.sync()
    assert (ws.numpy()[nb:] == 7).all()
    want, products = lo.gated(x, w, "silu")
    _near(pre.numpy(), products, TOL[dtype])
    _near(h.numpy(), want, TOL[dtype])
    nb = lib.d8_matmul_gated_scratch_bytes(dt, 1, rows, inner, cols)
    ws = DeviceArray((max(nb, 16),), np.uint8)
    (dxr, dxp), (dwr, dwp) = put(np.zeros_like(x), off[1]), put(np.zeros_like(w), off[0])
    check(lib.d8_matmul_gated_grad(dt, xp, dxp, rows, inner, wp, dwp, cols, 0, pre.ptr, gp, 3, ws.ptr, nb, None))
    capi.sync()
    wx, ww = lo.gated_grad(x, w, pre.numpy(), dh, "silu")
    for room, at, want in ((dxr, off[1], wx), (dwr, off[0], ww)):
        got = room.numpy()
        assert np.isnan(got[:at]).all() and np.isnan(got[-8:]).all()
        _near(got[at:-8].reshape(want.shape), want, TOL[dtype])
