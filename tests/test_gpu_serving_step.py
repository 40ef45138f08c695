"""A layer's half served in 8 bits, as a program runs it: norm of the rows, their codes, the products for queries, keys and values, rotation, the cache's new
tokens, attention over it, codes again and the product back.  Each step against its definition in 64 bits on what the step before left, at that step's
own tolerance (test_gpu_layer_norm.py, test_gpu_matmul_int8.py, test_gpu_cache.py); and the whole of it captured and replayed, the bits of the eager run."""
import ctypes

import numpy as np
import pytest

import layer_oracle as lo
import serving_oracle as so
from test_gpu_cache import TOL, _near as attention_near, _starts, _table
from test_gpu_layer_norm import _forward_terms, _within
from test_gpu_matmul_int8 import _near as product_near, _padded
from util import f, rng

pytestmark = pytest.mark.gpu
WIDTH, H, G, D = 192, 6, 2, 32


class _Layer:
    def __init__(self, dtype, longest):
        from deep8_amd import capi, ops
        self.capi, self.lib, self.ops, self.dtype, r = capi, capi.init(), ops, dtype, rng(21)
        self.dt, n = capi.dtype_id(dtype), lambda *s: r.standard_normal(s)  # noqa: E731
        self.norm, self.bias = (1 + 0.2 * n(WIDTH)).astype(dtype), (0.2 * n(WIDTH)).astype(dtype)
        self.w = {"q": n(WIDTH, H * D), "k": n(WIDTH, G * D), "v": n(WIDTH, G * D), "o": n(H * D, WIDTH)}
        self.w = {name: ops.quantize_columns((w * w.shape[0] ** -0.5).astype(dtype)) for name, w in self.w.items()}
        self.table, pages = _table(longest, r)
        self.angles = lo.table(max(longest), D).astype(np.float32)
        self.cache, self.want = ops.PagedCache(pages, G, D), so.Cache(pages, G, D)
        a = capi.DeviceArray.from_numpy
        self.d = {"norm": a(self.norm), "bias": a(self.bias), "angles": a(self.angles), "table": a(self.table)}
        for name, (codes, scales) in self.w.items():
            self.d["w" + name], self.d["s" + name] = a(codes), a(scales)

    def room(self, tokens, sequences):
        capi, lib = self.capi, self.lib
        e = lambda *s, t=self.dtype: capi.DeviceArray(s, t)  # noqa: E731
        pitch, pitch_o = lib.d8_int8_pitch(WIDTH), lib.d8_int8_pitch(H * D)
        b = {"x": e(tokens, WIDTH), "n": e(tokens, WIDTH), "nc": e(tokens, pitch, t=np.int8), "ns": e(tokens, t=np.float32), "q": e(tokens, H * D), "k": e(tokens, G * D),
             "v": e(tokens, G * D), "o": e(tokens, H * D), "oc": e(tokens, pitch_o, t=np.int8), "os": e(tokens, t=np.float32), "y": e(tokens, WIDTH), "lse": e(H, tokens, t=np.float32),
             "starts": e(sequences + 1, t=np.int32), "lengths": e(sequences, t=np.int32), "at": e(tokens, t=np.int32)}
        need = [lib.d8_matmul_int8_scratch_bytes(tokens, WIDTH, H * D), lib.d8_matmul_int8_scratch_bytes(tokens, H * D, WIDTH),
                lib.d8_attention_cache_scratch_bytes(self.dt, sequences, tokens, self.table.shape[1], H, G, D)]
        b["scratch"] = e(max(need), t=np.uint8)
        return b

    def step(self, b, cache, stream=None):
        """the calls, on one stream, without a look at what they leave"""
        lib, d, dt, (tokens, _), sequences = self.lib, self.d, self.dt, b["x"].shape, b["lengths"].shape[0]
        p = {name: a.ptr for name, a in b.items()}
        scratch = (p["scratch"], b["scratch"].nbytes)
        check = self.capi.check
        check(lib.d8_layer_norm(dt, p["x"], WIDTH, d["norm"].ptr, d["bias"].ptr, p["n"], WIDTH, tokens, WIDTH, 1e-5, stream))
        check(lib.d8_quantize_rows(dt, p["n"], WIDTH, tokens, WIDTH, p["nc"], p["ns"], stream))
        for name, cols in (("q", H * D), ("k", G * D), ("v", G * D)):
            check(lib.d8_matmul_int8(dt, p["nc"], p["ns"], tokens, WIDTH, d["w" + name].ptr, d["s" + name].ptr, cols, p[name], cols, *scratch, stream))
        check(lib.d8_head_norm_rotary(dt, p["q"], H * D, H, None, p["q"], H * D, p["k"], G * D, G, None, p["k"], G * D, tokens, D, 0, 0.0, p["at"], d["angles"].ptr,
                                      len(self.angles), D, 0, stream))
        where = (p["starts"], p["lengths"], d["table"].ptr, sequences, tokens, self.table.shape[1], cache.pages)
        check(lib.d8_cache_append(dt, p["k"], G * D, p["v"], G * D, *cache._state(), *where, G, D, stream))
        check(lib.d8_attention_cache(dt, p["q"], H * D, *cache._state(), p["o"], H * D, p["lse"], *where, H, G, D, D ** -0.5, 1, *scratch, stream))
        check(lib.d8_quantize_rows(dt, p["o"], H * D, tokens, H * D, p["oc"], p["os"], stream))
        check(lib.d8_matmul_int8(dt, p["oc"], p["os"], tokens, H * D, d["wo"].ptr, d["so"].ptr, WIDTH, p["y"], WIDTH, *scratch, stream))

    def feed(self, b, x, new, held):
        b["x"].copy_from(x), b["starts"].copy_from(_starts(new)), b["lengths"].copy_from(held)
        b["at"].copy_from(np.concatenate([np.arange(h - n, h) for n, h in zip(new, held)]))

    def check(self, b, new, held):
        self.capi.sync()
        g, dtype = {name: a.numpy() for name, a in b.items()}, self.dtype
        n, u = so.layer_norm(g["x"], self.norm, self.bias, 1e-5)
        _within(g["n"], n, _forward_terms(u, self.norm, self.bias), 32, dtype)
        codes, scales = so.quantize(g["n"])
        assert np.array_equal(g["nc"], _padded(codes, g["nc"].shape[1])) and np.array_equal(g["ns"], scales)
        at = np.concatenate([np.arange(h - m, h) for m, h in zip(new, held)])
        for name, heads in (("q", H), ("k", G)):
            product = so.matmul_int8(g["nc"], g["ns"], *self.w[name]).astype(dtype)
            turned = lo.norm_rotary(product.reshape(-1, heads, D), None, self.angles, at, D, False, False)
            # the product's rounding and the turn's: 2^-11 each of both elements of a pair (half), 4 and 3 roundings of 2^-24 (single)
            assert np.abs(f(g[name]) - turned.reshape(g[name].shape)).max() <= (4 * 2.0 ** -11 if dtype == np.float16 else 16 * 2.0 ** -24) * np.abs(turned).max()
        product_near(g["v"], so.matmul_int8(g["nc"], g["ns"], *self.w["v"]), dtype)
        tokens = len(at)
        self.want.append(g["k"].reshape(tokens, G, D), g["v"].reshape(tokens, G, D), _starts(new), held, self.table)
        values = [np.nan_to_num(self.want.codes[name] * self.want.scales[name][..., None, None]) for name in "kv"]
        o, lse = so.attention_cache(g["q"].reshape(tokens, H, D), *values, _starts(new), held, self.table, self.cache.pages, D ** -0.5, True)
        attention_near(g["o"].reshape(tokens, H, D), o, TOL[dtype])
        assert np.abs(g["lse"] - lse).max() <= 1e-5 * max(1, np.abs(lse).max())
        codes, scales = so.quantize(g["o"])
        assert np.array_equal(g["oc"], _padded(codes, g["oc"].shape[1])) and np.array_equal(g["os"], scales)
        product_near(g["y"], so.matmul_int8(g["oc"], g["os"], *self.w["o"]), dtype)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_a_layer_step_by_step(dtype):
    """a prompt, its next part, and tokens one by one"""
    layer, r = _Layer(dtype, [260, 71, 130]), rng(22)
    held = np.zeros(3, np.int64)
    for new in ([200, 3, 120], [57, 64, 7], [1, 1, 1], [1, 1, 1], [1, 2, 1]):
        held += new
        b = layer.room(sum(new), 3)
        layer.feed(b, (2 * r.standard_normal((sum(new), WIDTH))).astype(dtype), new, held)
        layer.step(b, layer.cache)
        layer.check(b, new, held)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_a_layer_captured_and_replayed(dtype):
    """one graph for every step of decoding; lengths, places and rows change between the replays, an eager layer runs beside them"""
    from deep8_amd import capi
    live, eager, r = _Layer(dtype, [150, 90]), _Layer(dtype, [150, 90]), rng(23)
    held, first = np.array([120, 64], np.int64), [120, 64]
    x = r.standard_normal((184, WIDTH)).astype(dtype)
    for layer in (live, eager):
        b = layer.room(184, 2)
        layer.feed(b, x, first, held)
        layer.step(b, layer.cache)
        capi.sync()
    b, e = live.room(2, 2), eager.room(2, 2)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    capi.check(live.lib.d8_stream_create(ctypes.byref(stream)))
    capi.check(live.lib.d8_graph_begin(stream))
    live.step(b, live.cache, stream)
    capi.check(live.lib.d8_graph_end(stream, ctypes.byref(graph)))
    for _ in range(4):
        held = held + 1
        x = r.standard_normal((2, WIDTH)).astype(dtype)
        live.feed(b, x, [1, 1], held), eager.feed(e, x, [1, 1], held)
        capi.check(live.lib.d8_graph_launch(graph, stream))
        capi.sync(stream)
        eager.step(e, eager.cache)
        capi.sync()
        assert all(np.array_equal(b[name].numpy(), e[name].numpy()) for name in ("n", "nc", "ns", "q", "k", "v", "o", "lse", "oc", "os", "y"))
        for name in ("k_codes", "v_codes", "k_scales", "v_scales"):
            assert np.array_equal(getattr(live.cache, name).numpy(), getattr(eager.cache, name).numpy(), equal_nan=True)
    capi.check(live.lib.d8_graph_destroy(graph))
    capi.check(live.lib.d8_stream_destroy(stream))


def test_two_layers_at_once():
    """two caches served on two streams, calls of both on their way together: the bits of each alone"""
    from deep8_amd import capi
    layers, alone, r = [_Layer(np.float16, [260, 140]) for _ in range(2)], _Layer(np.float16, [260, 140]), rng(24)
    streams = [ctypes.c_void_p() for _ in layers]
    for s in streams:
        capi.check(layers[0].lib.d8_stream_create(ctypes.byref(s)))
    calls, held = [], np.zeros(2, np.int64)
    for new in ([250, 130], [1, 1], [1, 2], [1, 1]):
        held = held + new
        x = r.standard_normal((2, sum(new), WIDTH)).astype(np.float16)
        rooms = [layer.room(sum(new), 2) for layer in layers]
        for layer, b, rows in zip(layers, rooms, x):
            layer.feed(b, rows, new, held)
        calls.append((new, held, x, rooms))
    capi.sync()
    for new, held, x, rooms in calls:
        for layer, b, s in zip(layers, rooms, streams):
            layer.step(b, layer.cache, s)
    for s in streams:
        capi.sync(s)
    for i in range(2):
        if i:
            alone = _Layer(np.float16, [260, 140])
        for new, held, x, rooms in calls:
            b = alone.room(sum(new), 2)
            alone.feed(b, x[i], new, held)
            alone.step(b, alone.cache)
            capi.sync()
            assert all(np.array_equal(b[name].numpy(), rooms[i][name].numpy()) for name in ("n", "nc", "q", "k", "v", "o", "lse", "oc", "y"))
    for s in streams:
        capi.check(layers[0].lib.d8_stream_destroy(s))
