"""d8_matmul_gated and its gradient against the formulas in 64 bits, within the framework's tolerances: 1e-5 in Float32 and 2e-3 in Float16
(roundings to half of at most 2^-11: the result's, and on the way back that of the gate's and the factor's gradients).  pre alone is a
plain product, whose Float16 rounding is half of that."""
import numpy as np
import pytest

import layer_oracle as lo
from util import FP16_TOL, FP32_TOL, f, rel_fro, rng

pytestmark = pytest.mark.gpu
TOL = {np.float16: FP16_TOL, np.float32: FP32_TOL}

SIZES = [
    # rows, inner, cols
    (1, 1, 1), (1, 64, 8), (1, 1000, 999), (2, 512, 1024), (3, 200, 72), (8, 2048, 96), (16, 136, 640), (17, 64, 264), (31, 300, 130), (64, 256, 256),
    (100, 100, 100), (128, 64, 64), (129, 33, 65), (256, 512, 128), (300, 130, 520), (257, 72, 200), (512, 256, 1024), (777, 100, 135), (1024, 192, 640),
    (1, 4096, 64), (5, 5000, 40), (4, 8, 4096), (33, 96, 72), (64, 1031, 520), (60, 2000, 24),
    (4096, 64, 1536), (4100, 128, 1544), (8200, 192, 1288), (256, 64, 24576),  # large tiles, more of them than compute units, moved back inside
]


def _near(got, want, tol):
    got, want = f(got).astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape and rel_fro(got, want) <= tol
    e, n = np.linalg.norm(got - want, axis=1), np.linalg.norm(want, axis=1)
    assert (e <= 4 * tol * (n + n.mean())).all()


def _inputs(rows, inner, cols, dtype):
    r = rng(rows + 3 * inner + 5 * cols)
    x, w = r.standard_normal((rows, inner)).astype(dtype), (r.standard_normal((inner, 2 * cols)) * inner ** -0.5).astype(dtype)
    return x, w, r.standard_normal((rows, cols)).astype(dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("size", SIZES)
def test_forward_and_gradient(size, dtype):
    from deep8_amd import ops
    act = ["silu", "gelu", "relu", "sigmoid"][sum(size) % 4]
    x, w, dh = _inputs(*size, dtype)
    want, pre = lo.gated(x, w, act)
    got, got_pre = ops.matmul_gated(x, w, act)
    _near(got_pre, pre, TOL[dtype])
    _near(got, want, TOL[dtype])
    alone, none = ops.matmul_gated(x, w, act, keep=False)
    assert none is None and np.array_equal(alone, got)
    dx, dw = ops.matmul_gated_grad(x, w, got_pre, dh, act)
    wx, ww = lo.gated_grad(x, w, got_pre, dh, act)
    _near(dx, wx, TOL[dtype])
    _near(dw, ww, TOL[dtype])
    sx, sw = ops.matmul_gated_grad(x, w, got_pre, dh, act, into=(np.ones_like(x), np.ones_like(w)))
    _near(sx, wx + 1, 2 * TOL[dtype])
    _near(sw, ww + 1, 2 * TOL[dtype])


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_gates_far_from_zero(act, dtype):
    """gates of -300 .. 300: nothing overflows on the way to 0 or to the gate itself"""
    from deep8_amd import ops
    g = np.linspace(-300, 300, 64).astype(dtype)
    w = np.concatenate([g, np.ones(64, dtype)])[None]
    x, dh = np.ones((3, 1), dtype), np.ones((3, 64), dtype)
    want, _ = lo.gated(x, w, act)
    got, pre = ops.matmul_gated(x, w, act)
    assert np.abs(f(got) - want).max() <= 300 * TOL[dtype]
    dx, dw = ops.matmul_gated_grad(x, w, pre, dh, act)
    wx, ww = lo.gated_grad(x, w, pre, dh, act)
    assert np.isfinite(f(dx)).all() and np.abs(f(dw) - ww).max() <= 1000 * TOL[dtype] and np.abs(f(dx) - wx).max() <= TOL[dtype] * np.abs(ww * f(w)).sum()


@pytest.mark.parametrize("rows", [1, 40, 300])
def test_what_is_no_number_stays_in_its_row_and_column(rows):
    from deep8_amd import ops
    x, w, _ = _inputs(rows, 128, 192, np.float16)
    want, _ = lo.gated(x, w, "silu")
    x[rows // 2, 5] = np.nan
    w[3, 7] = np.inf
    got, _ = ops.matmul_gated(x, w, "silu")
    rest = np.ones(got.shape, bool)
    rest[rows // 2], rest[:, 7] = False, False
    assert np.isnan(f(got[rows // 2])).all()
    assert np.isfinite(f(got)[rest]).all() and rel_fro(f(got)[rest], want[rest]) <= FP16_TOL if rest.any() else True


def test_stream_and_graph():
    import ctypes
    from deep8_amd import capi, ops
    lib = capi.init()
    x, w, _ = _inputs(2, 4096, 512, np.float16)
    want, _ = ops.matmul_gated(x, w, keep=False)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    capi.check(lib.d8_stream_create(ctypes.byref(stream)))
    a, b, h = capi.DeviceArray.from_numpy(x), capi.DeviceArray.from_numpy(w), capi.DeviceArray.from_numpy(np.zeros_like(want))
    nb = lib.d8_matmul_gated_scratch_bytes(capi.FLOAT16, 0, 2, 4096, 512)
    ws = capi.DeviceArray((max(nb, 16),), np.uint8)
    capi.check(lib.d8_graph_begin(stream))
    rc = lib.d8_matmul_gated(capi.FLOAT16, a.ptr, 2, 4096, b.ptr, 512, 0, None, h.ptr, ws.ptr, nb, stream)
    capi.check(lib.d8_graph_end(stream, ctypes.byref(graph)))
    capi.check(rc)
    for _ in range(3):
        h.copy_from(np.zeros_like(want))
        capi.check(lib.d8_graph_launch(graph, stream))
        capi.sync(stream)
        assert np.array_equal(h.numpy(), want)
    capi.check(lib.d8_graph_destroy(graph))
    capi.check(lib.d8_stream_destroy(stream))


def test_refusals():
    from deep8_amd import capi, ops
    x, w = np.zeros((2, 8), np.float32), np.zeros((8, 8), np.float32)
    with pytest.raises(capi.Deep8HipError):
        ops.matmul_gated(x.astype(np.float64), w.astype(np.float64))
    lib = capi.init()
    d = capi.DeviceArray((8, 8))
    call = lambda rows=2, inner=8, cols=4, act=0, x=d.ptr: lib.d8_matmul_gated(capi.FLOAT32, x, rows, inner, d.ptr, cols, act, None, d.ptr, None, 0, None)  # noqa: E731
    assert call(rows=0) == call(inner=0) == call(cols=-1) == call(act=4) == call(act=-1) == call(x=None) == 10001
    assert lib.d8_matmul_gated_grad(capi.FLOAT32, d.ptr, d.ptr, 2, 8, d.ptr, d.ptr, 4, 0, d.ptr, d.ptr, 3, None, 0, None) == 10001
    assert b"scratch" in lib.d8_last_error()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("size", [(65, 1030, 37), (130, 2056, 200), (777, 600, 1351)])
def test_tiles_in_parts(size, dtype):
    """few tiles, or a few left over, over a long inner axis: parts of the sums meet in a second launch"""
    from deep8_amd import ops
    x, w, _ = _inputs(*size, dtype)
    want, pre = lo.gated(x, w, "silu")
    got, got_pre = ops.matmul_gated(x, w, "silu")
    _near(got_pre, pre, TOL[dtype])
    _near(got, want, TOL[dtype])
    again, _ = ops.matmul_gated(x, w, "silu")
    assert np.array_equal(got, again)
