"""d8_quantize_rows, d8_quantize_columns and d8_matmul_int8 against their definitions in 64 bits.

Codes and scales have one right value: equal.  Products: the sum is exact; it is rounded to fp32, as are the scales' product and the result, 2^-24 each,
and then to the element type, half a step.  4 * 2^-24 and 2^-11 (half; its smallest numbers are 2^-24 apart) cover them, element by element."""
import ctypes

import numpy as np
import pytest

import serving_oracle as so
from util import f, rng

SIZES = [(1, 1), (3, 7), (2, 127), (2, 128), (5, 129), (1, 512), (9, 520), (33, 1000), (4, 1023), (3, 2048), (3, 4096), (2, 8192), (2, 8200), (2, 16384), (2, 16390), (2, 20001),
         (600, 96)]


def _x(rows, cols, dtype, seed):
    r = rng(seed)
    return (r.standard_normal((rows, cols)) * (1 + 7 * (r.random(cols) < 0.02)) * np.exp2(r.integers(-6, 6, (rows, 1)))).astype(dtype)


def _padded(codes, pitch):
    return np.pad(codes, ((0, 0), (0, pitch - codes.shape[1])))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_codes(rows, cols, dtype):
    from deep8_amd import ops
    x = _x(rows, cols, dtype, rows + cols)
    want, scales = so.quantize(x)
    for pad in (0, 1, 8):
        got, s = ops.quantize_rows(x, pad)
        assert np.array_equal(s, scales) and np.array_equal(got, _padded(want, got.shape[1]))
        got, s = ops.quantize_columns(np.ascontiguousarray(x.T), pad)
        assert np.array_equal(s, scales) and np.array_equal(got, _padded(want, got.shape[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_quotients_next_to_a_half(dtype):
    """rows whose scale is a whole power of two, values at halves of a step and the numbers of the type on both sides of each; rows of other
    scales, values next to every half"""
    from deep8_amd import ops
    half = np.arange(-126.5, 127, 1.0)
    rows = []
    for top in (127.0, 127 * 2.0 ** -9, 127 * 2.0 ** 5, 100.0, 3.1, 0.777):
        top = dtype(top)
        step = np.float32(top) / np.float32(127)
        at = (half * np.float64(step)).astype(dtype)
        row = np.concatenate([at, np.nextafter(at, dtype(np.inf)), np.nextafter(at, dtype(-np.inf))])
        rows.append(np.concatenate([[top], row[np.abs(row) < top]]))
    width = max(map(len, rows))
    x = np.stack([np.pad(r, (0, width - len(r))) for r in rows]).astype(dtype)
    want, scales = so.quantize(x)
    for got, s in (ops.quantize_rows(x), ops.quantize_columns(np.ascontiguousarray(x.T))):
        assert np.array_equal(s, scales) and np.array_equal(got, _padded(want, got.shape[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("cols", [40, 20000])
def test_rows_of_zeros_of_the_smallest_and_of_no_numbers(cols, dtype):
    from deep8_amd import ops
    x = np.zeros((8, cols), dtype)
    x[1] = np.finfo(dtype).smallest_subnormal
    x[2] = np.finfo(dtype).max
    x[3] = -np.finfo(dtype).tiny
    x[4, 3], x[5, 5], x[6, 7] = np.nan, np.inf, -np.inf
    x[4, 8:11] = 1
    x[7] = -1
    want, scales = so.quantize(x)
    for got, s in (ops.quantize_rows(x), ops.quantize_columns(np.ascontiguousarray(x.T))):
        assert np.array_equal(s, scales, equal_nan=True) and np.array_equal(got, _padded(want, got.shape[1]))
    z = ops.matmul_int8(*ops.quantize_rows(x), *ops.quantize_rows(x), cols)
    bad = np.isnan(scales)
    assert np.isnan(z[bad]).all() and np.isnan(z[:, bad]).all()
    assert not z[0][~bad].any()


PRODUCTS = [(1, 1, 1), (1, 64, 31), (3, 200, 33), (4, 4096, 512), (16, 1000, 100), (17, 300, 64), (32, 2048, 70), (33, 130, 5), (64, 8192, 48), (5, 16, 9000), (2, 131071, 3),
            (65, 128, 65), (128, 4096, 128), (130, 1000, 257), (777, 1000, 1351), (200, 100, 4100), (2000, 700, 2050), (100, 20000, 70),
            (4, 16384, 130), (20, 8192, 100), (40, 8192, 1000), (32, 200, 9000), (50, 100, 9000)]


def _product(rows, inner, cols, seed):
    r, pitch = rng(seed), (inner + 127) // 128 * 128
    c = lambda n: _padded(r.integers(-128, 128, (n, inner), dtype=np.int8), pitch)  # noqa: E731
    return c(rows), np.exp(r.standard_normal(rows)).astype(np.float32) * 1e-2, c(cols), np.exp(r.standard_normal(cols)).astype(np.float32) * 1e-3


def _near(got, want, dtype):
    got = f(got).astype(np.float64)
    half, tiny = (2.0 ** -11, 2.0 ** -25) if dtype == np.float16 else (0.0, 0.0)
    big = np.abs(want) > 65504 if dtype == np.float16 else np.zeros(want.shape, bool)
    assert (np.abs(got - want) <= (half + 4 * 2.0 ** -24) * np.abs(want) + tiny)[~big].all()
    assert (np.isinf(got) | (np.abs(got) == 65504))[big].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,inner,cols", PRODUCTS)
def test_products(rows, inner, cols, dtype):
    from deep8_amd import ops
    x, xs, w, ws = _product(rows, inner, cols, rows + inner + cols)
    want = so.matmul_int8(x, xs, w, ws)
    for pad in (0, 1, 4):
        _near(ops.matmul_int8(x, xs, w, ws, inner, dtype, pad), want, dtype)


@pytest.mark.gpu
def test_all_extremes():
    """the largest sum there is, 128 * 128 * 131071, and its negative"""
    from deep8_amd import ops
    inner = 131071
    for rows in (2, 70):
        x = np.pad(np.full((rows, inner), -128, np.int8), ((0, 0), (0, 1)))
        w = x[:2].copy()
        w[1, :inner] = 127
        one = np.ones(rows, np.float32)
        _near(ops.matmul_int8(x, one, w, one[:2], inner), so.matmul_int8(x, one, w, one[:2]), np.float32)


# many rows and columns: whole tiles of 256, one row and column more, rows of z that start anywhere, one step of the reduction, odd counts of steps
WIDE = [(4096, 128, 4096, 0), (4097, 384, 3600, 8), (3600, 1000, 4097, 0), (5000, 256, 3333, 3), (300, 640, 60000, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,inner,cols,pad", WIDE)
def test_wide_products(rows, inner, cols, pad, dtype):
    """each of a hundred rows and columns in full, the last ones among them"""
    from deep8_amd import ops
    x, xs, w, ws = _product(rows, inner, cols, rows)
    got = ops.matmul_int8(x, xs, w, ws, inner, dtype, pad)
    r = rng(1)
    for n, axis in ((rows, 0), (cols, 1)):
        pick = np.unique(np.concatenate([[0, n - 1, n - 2, 255, 256, n - 257], r.integers(0, n, 100)]))
        part = so.matmul_int8(x[pick], xs[pick], w, ws) if axis == 0 else so.matmul_int8(x, xs, w[pick], ws[pick])
        _near(np.take(got, pick, axis), part, dtype)


@pytest.mark.gpu
def test_a_product_with_its_quantised_operands_is_near_the_product():
    """each code is off by half a step at most: |z - x w| <= sum |x| step_w / 2 + |w| step_x / 2 + step_x step_w / 4, and the fp32 roundings"""
    from deep8_amd import ops
    r = rng(3)
    x, w = r.standard_normal((37, 300)).astype(np.float32), r.standard_normal((300, 41)).astype(np.float32)
    xc, xs = ops.quantize_rows(x)
    wc, ws = ops.quantize_columns(w)
    z = ops.matmul_int8(xc, xs, wc, ws, 300)
    bound = np.abs(x).sum(1)[:, None] * ws / 2 + np.abs(w).sum(0) * xs[:, None] / 2 + 300 * xs[:, None] * ws / 4
    assert (np.abs(z - x.astype(np.float64) @ w) <= 1.0001 * bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,inner,cols", [(4, 4096, 512), (4, 16384, 512), (300, 1000, 130), (4096, 256, 4096)])
def test_captured_and_replayed(rows, inner, cols):
    from deep8_amd import capi, ops
    lib = capi.init()
    x, w = _x(rows, inner, np.float16, 1), _x(inner, cols, np.float16, 2)
    eager = lambda: ops.matmul_int8(*ops.quantize_rows(x), *ops.quantize_columns(w), inner, np.float16)  # noqa: E731
    want = eager()
    pitch = lib.d8_int8_pitch(inner)
    d = [capi.DeviceArray.from_numpy(a) for a in (x, w)]
    xc, wc, z = capi.DeviceArray((rows, pitch), np.int8), capi.DeviceArray((cols, pitch), np.int8), capi.DeviceArray((rows, cols), np.float16)
    xs, ws = capi.DeviceArray((rows,)), capi.DeviceArray((cols,))
    nb = lib.d8_matmul_int8_scratch_bytes(rows, inner, cols)
    scratch = capi.DeviceArray((max(nb, 16),), np.uint8)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    capi.check(lib.d8_stream_create(ctypes.byref(stream)))
    capi.check(lib.d8_graph_begin(stream))
    rcs = [lib.d8_quantize_rows(capi.FLOAT16, d[0].ptr, inner, rows, inner, xc.ptr, xs.ptr, stream),
           lib.d8_quantize_columns(capi.FLOAT16, d[1].ptr, cols, inner, cols, wc.ptr, ws.ptr, stream),
           lib.d8_matmul_int8(capi.FLOAT16, xc.ptr, xs.ptr, rows, inner, wc.ptr, ws.ptr, cols, z.ptr, cols, scratch.ptr, nb, stream)]
    capi.check(lib.d8_graph_end(stream, ctypes.byref(graph)))
    assert rcs == [0, 0, 0]
    for _ in range(3):
        for o in (xc, wc, z, xs, ws):
            o.copy_from(np.full(o.shape, 7, o.dtype))
        capi.check(lib.d8_graph_launch(graph, stream))
        capi.sync(stream)
        assert np.array_equal(z.numpy(), want)
        eager()
    capi.check(lib.d8_graph_destroy(graph))
    capi.check(lib.d8_stream_destroy(stream))


@pytest.mark.gpu
def test_nothing_to_do():
    from deep8_amd import ops
    codes, scales = ops.quantize_rows(np.zeros((0, 24), np.float32))
    assert codes.shape == (0, 128) and scales.shape == (0,)
    codes, scales = ops.quantize_columns(np.zeros((24, 0), np.float32))
    assert codes.shape == (0, 128)
    one = np.zeros((3, 128), np.int8), np.ones(3, np.float32)
    assert ops.matmul_int8(codes, scales, *one, 24).shape == (0, 3) and ops.matmul_int8(*one, codes, scales, 24).shape == (3, 0)


@pytest.mark.gpu
def test_more_tiles_of_columns_than_a_launch_has_along_an_axis():
    """32768 tiles of 64 columns and two more, some rows too many for the kernel of few; results at both sides of the turn and at random places"""
    from deep8_amd import capi
    lib, r, rows, cols = capi.init(), rng(41), 65, 32768 * 64 + 70
    w, x = np.zeros((cols, 128), np.int8), np.zeros((rows, 128), np.int8)
    w[:, 0], x[:, 0] = r.integers(-127, 128, cols), r.integers(-127, 128, rows)
    xs, ws = np.exp2(r.integers(-4, 3, rows)).astype(np.float32), np.exp2(r.integers(-4, 3, cols)).astype(np.float32)
    d = [capi.DeviceArray.from_numpy(a) for a in (x, xs, w, ws)]
    z = capi.DeviceArray((rows, cols), np.float16)
    capi.check(lib.d8_matmul_int8(capi.FLOAT16, d[0].ptr, d[1].ptr, rows, 1, d[2].ptr, d[3].ptr, cols, z.ptr, cols, None, 0, None))
    capi.sync()
    at = np.r_[0:70, 32768 * 64 - 70:cols, r.integers(0, cols, 500)]
    want = (x[:, :1].astype(np.float64) * xs[:, None]) * (w[at, 0].astype(np.float64) * ws[at])
    with np.errstate(over="ignore"):  # (some are more than half holds)
        assert np.array_equal(z.numpy()[:, at], want.astype(np.float16))


def test_refusals():
    """(refused before anything is launched: the tensors need not be there, nor a device)"""
    from deep8_amd import capi
    lib, p = capi.load(), 64
    assert [lib.d8_int8_pitch(n) for n in (-1, 0, 1, 128, 129, 131071, 131072)] == [0, 0, 128, 128, 256, 131072, 0]

    def refused(fn, good, cases, code=10001):
        for i, v in cases:
            a = list(good)
            a[i] = v
            assert fn(*a) == code, (fn.__name__, i, v)
    rows = (capi.FLOAT16, p, 8, 4, 8, p, p, None)
    for fn in (lib.d8_quantize_rows, lib.d8_quantize_columns):
        refused(fn, rows, [(1, None), (2, 7), (3, -1), (4, -1), (5, None), (5, 72), (6, None)])
        refused(fn, rows, [(0, capi.FLOAT64), (0, 0)], 10002)
    refused(lib.d8_quantize_rows, rows, [(4, 0), (4, 131072)])
    refused(lib.d8_quantize_columns, rows, [(3, 0), (3, 131072)])
    product = (capi.FLOAT16, p, p, 4, 16384, p, p, 8, p, 8, p, 1 << 40, None)
    assert lib.d8_matmul_int8_scratch_bytes(4, 16384, 8) > 0
    refused(lib.d8_matmul_int8, product, [(1, None), (1, 72), (2, None), (3, -1), (4, 0), (4, 131072), (5, None), (5, 65), (6, None), (7, -1), (8, None), (9, 7), (10, None), (10, 72),
                                          (11, 0)])
    refused(lib.d8_matmul_int8, product, [(0, capi.FLOAT64)], 10002)
    for rows, cols in ((1, 1 << 28), (100, 1 << 30)):  # more than the threads of a launch
        assert lib.d8_matmul_int8(capi.FLOAT16, p, p, rows, 128, p, p, cols, p, cols, p, 1 << 40, None) == 10001
    assert lib.d8_matmul_int8_scratch_bytes(4, 131072, 8) == 0 and lib.d8_matmul_int8_scratch_bytes(-1, 8, 8) == 0
