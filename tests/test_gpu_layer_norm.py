"""d8_layer_norm and d8_layer_norm_grad against the formulas in 64 bits.

Tolerances, element by element.  HALF: the result's own rounding, half a step of its type.  Before it everything is fp32 (steps of 2^-23, half a
step E = 2^-24): an element's distance from the mean is good to E of itself and, by the mean, to a few E of the spread; the spread's square is a
sum of at most 16 terms a lane in a row, then 6 + 2 levels of lanes and waves: 24 roundings; the reciprocal of its root three more.  32 E of what is added up covers
it.  dx adds two more such sums: 64 E.  dw and db: a row's term as above, then sums of at most 20 rows a lane, 16 teams, 16 workgroups a wave and
16 waves (teams of 16 threads: a row, 32 teams, 9 workgroups, 16 waves): 68 roundings more, 128 E in all."""
import ctypes

import numpy as np
import pytest

import serving_oracle as so
from util import f, rng

HALF = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24}
E = 2.0 ** -24
TINY = {np.float16: 2.0 ** -25, np.float32: 0.0}  # half a step of the smallest numbers

# rows, cols, pad: teams of 16, 32, 64, 256, 512 and 1024 threads with 8 and 16 elements each, rows in 16-byte pieces and not, shorter than one, rows that no team holds
CASES = [(1, 1, 0), (3, 7, 1), (5, 64, 0), (2, 512, 8), (9, 520, 0), (33, 1000, 0), (3, 1024, 3), (7, 1025, 0), (5, 2048, 0), (3, 2056, 8), (6, 4096, 0),
         (2, 4097, 0), (3, 8192, 0), (2, 8200, 8), (3, 16384, 0), (2, 16384, 1), (3, 16385, 0), (2, 20000, 8), (700, 96, 0), (4099, 100, 0), (1030, 1000, 24),
         (700, 3, 0), (65, 8, 0), (33, 9, 1), (70, 128, 0), (33, 127, 1), (9, 129, 3), (301, 200, 0), (40, 256, 8), (33, 255, 1), (3, 257, 0), (4, 2047, 0), (300, 4095, 5), (2, 5120, 0), (3, 8191, 2), (2, 8193, 0), (2, 11111, 0)]


def _inputs(rows, cols, dtype, seed, shift=0.0):
    r = rng(seed)
    x = (2 * r.standard_normal((rows, cols)) + r.standard_normal((rows, 1)) + shift).astype(dtype)
    return x, (1 + 0.2 * r.standard_normal(cols)).astype(dtype), (0.2 * r.standard_normal(cols)).astype(dtype), r.standard_normal((rows, cols)).astype(dtype)


def _within(got, want, terms, n, dtype):
    got = f(got).astype(np.float64)
    assert got.shape == want.shape
    assert (np.abs(got - want) <= HALF[dtype] * np.abs(want) * 1.001 + n * E * terms + TINY[dtype]).all()


def _forward_terms(u, w, b):
    w = 1.0 if w is None else np.abs(f(w))
    return (np.abs(u) + 1) * w + (0 if b is None else np.abs(f(b)))


def _grad_terms(x, dy, w, epsilon):
    _, u = so.layer_norm(x, None, None, epsilon)
    x = np.asarray(x, np.float64)
    r = 1 / np.sqrt(x.var(-1, keepdims=True) + epsilon)
    wg = np.abs(f(dy) * (1 if w is None else f(w))).astype(np.float64)
    dx = r * (wg + wg.mean(-1, keepdims=True) + (np.abs(u) + 1) * (wg * (np.abs(u) + 1)).mean(-1, keepdims=True))
    return dx, (np.abs(f(dy)) * (np.abs(u) + 1)).sum(0), np.abs(f(dy)).sum(0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols,pad", CASES)
def test_forward_and_gradient(rows, cols, pad, dtype):
    from deep8_amd import ops
    x, w, b, dy = _inputs(rows, cols, dtype, rows + cols)
    for weight, bias in ((w, b), (None, None), (w, None)):
        y, u = so.layer_norm(x, weight, bias, 1e-5)
        _within(ops.layer_norm(x, weight, bias, pad=pad), y, _forward_terms(u, weight, bias), 32, dtype)
    assert np.array_equal(ops.layer_norm(x, w, b, pad=pad, in_place=True), ops.layer_norm(x, w, b, pad=pad))
    for weight in (w, None):
        want, terms = so.layer_norm_grad(x, dy, weight, 1e-5), _grad_terms(x, dy, weight, 1e-5)
        got = ops.layer_norm_grad(x, dy, weight, pad=pad)
        for g, v, t, n in zip(got, want, terms, (64, 128, 128)):
            _within(g, v, t, n, dtype)
        again = ops.layer_norm_grad(x, dy, weight, pad=pad)
        assert all(np.array_equal(p, q) for p, q in zip(got, again))
    old = [rng(5).standard_normal(a.shape).astype(dtype) for a in (x, w, b)]
    for g, v, t, o, n in zip(ops.layer_norm_grad(x, dy, w, pad=pad, into=old), so.layer_norm_grad(x, dy, w, 1e-5), _grad_terms(x, dy, w, 1e-5), old, (64, 128, 128)):
        _within(g, v + f(o), t + np.abs(f(o)), n, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1000, 1001, 4096, 20000])
def test_rows_far_from_zero(cols):
    """a mean of a thousand times the spread: the sum of squares less the square of the mean would leave nothing of it"""
    from deep8_amd import ops
    x, w, b, dy = _inputs(6, cols, np.float32, cols, shift=2000.0)
    y, u = so.layer_norm(x, w, b, 1e-5)
    _within(ops.layer_norm(x, w, b), y, _forward_terms(u, w, b), 32, np.float32)
    for g, v, t, n in zip(ops.layer_norm_grad(x, dy, w), so.layer_norm_grad(x, dy, w, 1e-5), _grad_terms(x, dy, w, 1e-5), (64, 128, 128)):
        _within(g, v, t, n, np.float32)


@pytest.mark.gpu
def test_rows_of_one_value_and_rows_that_are_no_numbers():
    from deep8_amd import ops
    x, w, b, dy = _inputs(5, 96, np.float32, 3)
    x[1], x[2, 5], x[3, 7] = 3.0, np.nan, np.inf
    y = ops.layer_norm(x, w, b)
    assert np.array_equal(y[1], b)  # no spread: the bias alone
    assert np.isnan(y[2]).all() and np.isnan(y[3]).all() and np.isfinite(y[[0, 1, 4]]).all()
    dx, dw, db = ops.layer_norm_grad(x, dy, w)
    assert np.isnan(dx[2]).all() and np.isnan(dx[3]).all() and np.isfinite(dx[[0, 1, 4]]).all()
    assert np.isnan(dw).all() and np.isfinite(db).all()


@pytest.mark.gpu
@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (False, False, False)])
def test_gradients_that_are_not_wanted(wanted):
    from deep8_amd import ops
    for cols in (130, 17000):
        x, w, b, dy = _inputs(20, cols, np.float32, 4)
        for got, want, wish in zip(ops.layer_norm_grad(x, dy, w, wanted=wanted), ops.layer_norm_grad(x, dy, w), wanted):
            assert np.array_equal(got, want) if wish else got is None


@pytest.mark.gpu
def test_gradient_against_differences():
    from deep8_amd import ops
    x, w, b, dy = _inputs(3, 40, np.float32, 9)
    dx, dw, db = ops.layer_norm_grad(x, dy, w)
    loss = lambda x, w, b: (so.layer_norm(x, w, b, 1e-5)[0] * dy).sum()  # noqa: E731
    step = 1e-4  # central differences: off by step^2 times a third derivative, 1e-8, and in 64 bits by 1e-16 / step
    for got, which in ((dx, 0), (dw, 1), (db, 2)):
        for i in np.ndindex(got.shape):
            p, q = ([np.asarray(a, np.float64).copy() for a in (x, w, b)] for _ in range(2))
            p[which][i] += step
            q[which][i] -= step
            assert abs((loss(*p) - loss(*q)) / (2 * step) - got[i]) <= 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["dx is dy", "dx is x"])
@pytest.mark.parametrize("cols", [96, 1001, 4096, 17000])
def test_gradient_over_an_input(which, cols):
    from deep8_amd import capi, ops
    lib = capi.init()
    x, w, _, dy = _inputs(300, cols, np.float32, 11)
    want = ops.layer_norm_grad(x, dy, w)[0]
    d = [capi.DeviceArray.from_numpy(a) for a in (x, dy, w)]
    over = d[1] if which == "dx is dy" else d[0]
    capi.check(lib.d8_layer_norm_grad(capi.FLOAT32, d[0].ptr, cols, d[2].ptr, d[1].ptr, cols, over.ptr, cols, None, None, 300, cols, 1e-5, 3, None, 0, None))
    capi.sync()
    assert np.array_equal(over.numpy(), want)


@pytest.mark.gpu
def test_no_rows():
    from deep8_amd import ops
    x = np.zeros((0, 24), np.float32)
    assert ops.layer_norm(x).shape == (0, 24)
    dx, dw, db = ops.layer_norm_grad(x, x)
    assert dx.shape == (0, 24) and not dw.any() and not db.any()
    old = (x, np.ones(24, np.float32), np.full(24, 2, np.float32))
    _, dw, db = ops.layer_norm_grad(x, x, into=old)
    assert (dw == 1).all() and (db == 2).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols", [(40, 96), (300, 1001), (1000, 4096), (5, 17000)])
def test_captured_and_replayed(rows, cols, dtype):
    """both directions on a stream of the caller's, captured: the bits of the eager calls at every replay, with eager calls of other sizes between them"""
    from deep8_amd import capi, ops
    lib = capi.init()
    code = capi.FLOAT16 if dtype == np.float16 else capi.FLOAT32
    x, w, b, dy = _inputs(rows, cols, dtype, rows)
    want = (ops.layer_norm(x, w, b), *ops.layer_norm_grad(x, dy, w))
    d = [capi.DeviceArray.from_numpy(a) for a in (x, w, b, dy)]
    out = [capi.DeviceArray.from_numpy(np.full(a.shape, 7, dtype)) for a in want]
    nb = lib.d8_layer_norm_grad_scratch_bytes(code, rows, cols)
    scratch = capi.DeviceArray((nb,), np.uint8)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    capi.check(lib.d8_stream_create(ctypes.byref(stream)))
    capi.sync()
    capi.check(lib.d8_graph_begin(stream))
    rcs = (lib.d8_layer_norm(code, d[0].ptr, cols, d[1].ptr, d[2].ptr, out[0].ptr, cols, rows, cols, 1e-5, stream),
           lib.d8_layer_norm_grad(code, d[0].ptr, cols, d[1].ptr, d[3].ptr, cols, out[1].ptr, cols, out[2].ptr, out[3].ptr, rows, cols, 1e-5, 3, scratch.ptr, nb, stream))
    capi.check(lib.d8_graph_end(stream, ctypes.byref(graph)))
    for rc in rcs:
        capi.check(rc)
    for _ in range(3):
        for o in out:
            o.copy_from(np.full(o.shape, 7, dtype))
        capi.check(lib.d8_graph_launch(graph, stream))
        capi.sync(stream)
        assert all(np.array_equal(o.numpy(), a) for o, a in zip(out, want))
        ops.layer_norm_grad(x[: rows // 2], dy[: rows // 2], w)
    capi.check(lib.d8_graph_destroy(graph))
    capi.check(lib.d8_stream_destroy(stream))


def test_refusals():
    """(refused before anything is launched: the tensors need not be there, nor a device)"""
    from deep8_amd import capi
    lib, p = capi.load(), 64
    ok = (capi.FLOAT32, p, 8, p, p, p, 8, 4, 8, 1e-5, None)

    def forward(**kw):
        a = list(ok)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return lib.d8_layer_norm(*a)
    assert forward(_0=capi.FLOAT64) == 10002 and forward(_0=0) == 10002
    for bad in (dict(_1=None), dict(_5=None), dict(_2=7), dict(_6=7), dict(_7=-1), dict(_8=0), dict(_8=1 << 30, _2=1 << 31, _6=1 << 31), dict(_9=-1.0), dict(_9=float("nan"))):
        assert forward(**bad) == 10001, bad
    nb = 1 << 40
    good = (capi.FLOAT16, p, 8, p, p, 8, p, 8, p, p, 4, 8, 1e-5, 3, p, nb, None)

    def grad(**kw):
        a = list(good)
        for k, v in kw.items():
            a[int(k[1:])] = v
        return lib.d8_layer_norm_grad(*a)
    assert grad(_0=capi.FLOAT64) == 10002
    for bad in (dict(_1=None), dict(_4=None), dict(_2=7), dict(_5=7), dict(_7=7), dict(_10=-1), dict(_11=0), dict(_14=None), dict(_15=15), dict(_14=72)):
        assert grad(**bad) == 10001, bad
    assert lib.d8_layer_norm_grad_scratch_bytes(capi.FLOAT64, 4, 8) == 0 and lib.d8_layer_norm_grad_scratch_bytes(capi.FLOAT32, -1, 8) == 0
