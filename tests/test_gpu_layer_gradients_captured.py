"""The gradient calls of a transformer layer on a stream of the caller's, captured and replayed: the bits of the eager call, every time.  And
d8_head_norm_rotary_grad with the gradients of its inputs written over those of its outputs."""
import ctypes

import numpy as np
import pytest

from test_gpu_attention import _inputs as attention_inputs, _starts
from test_gpu_head_norm_rotary import CASES as ROTARY_CASES, _inputs as rotary_inputs
from test_gpu_matmul_gated import _inputs as gated_inputs

pytestmark = pytest.mark.gpu


def _replayed(call, outputs, want, between):
    """`call` captured on a stream of its own, replayed three times over outputs that were overwritten"""
    from deep8_amd import capi
    lib = capi.init()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    capi.check(lib.d8_stream_create(ctypes.byref(stream)))
    capi.check(lib.d8_graph_begin(stream))
    rc = call(stream)
    capi.check(lib.d8_graph_end(stream, ctypes.byref(graph)))
    capi.check(rc)
    for _ in range(3):
        for o in outputs:
            o.copy_from(np.full(o.shape, 7, o.dtype))
        capi.check(lib.d8_graph_launch(graph, stream))
        capi.sync(stream)
        assert all(np.array_equal(o.numpy(), w) for o, w in zip(outputs, want))
        between()
    capi.check(lib.d8_graph_destroy(graph))
    capi.check(lib.d8_stream_destroy(stream))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("nq,D", [([20, 9], 64), ([900, 300], 128)])
def test_attention_grad(nq, D, dtype):
    from deep8_amd import capi, ops
    lib, H, G = capi.init(), 8, 2
    q, k, v, do = attention_inputs(nq, nq, H, G, D, dtype, 90)
    s = _starts(nq)
    o, lse = ops.attention(q, k, v, s, s, D ** -0.5)
    eager = lambda: ops.attention_grad(q, k, v, o, lse, do, s, s, D ** -0.5)  # noqa: E731
    want = eager()
    d = [capi.DeviceArray.from_numpy(a) for a in (q, k, v, o, lse, do, s)]
    out = [capi.DeviceArray(a.shape, dtype) for a in want]
    n = (2, sum(nq), sum(nq), H, G, D)
    nb = lib.d8_attention_scratch_bytes(capi.dtype_id(dtype), 1, *n, 1)
    ws = capi.DeviceArray((nb,), np.uint8)
    q_row, k_row = H * D, G * D

    def call(stream):
        return lib.d8_attention_grad(capi.dtype_id(dtype), d[0].ptr, q_row, d[1].ptr, k_row, d[2].ptr, k_row, d[3].ptr, q_row, d[4].ptr, d[5].ptr, q_row, out[0].ptr,
                                     q_row, out[1].ptr, k_row, out[2].ptr, k_row, d[6].ptr, d[6].ptr, *n, D ** -0.5, 1, 7, ws.ptr, nb, stream)
    _replayed(call, out, want, eager)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("size", [(3, 200, 72), (777, 104, 135), (512, 256, 1024)])
def test_matmul_gated_grad(size, dtype):
    from deep8_amd import capi, ops
    lib = capi.init()
    rows, inner, cols = size
    x, w, dh = gated_inputs(*size, dtype)
    _, pre = ops.matmul_gated(x, w)
    eager = lambda: ops.matmul_gated_grad(x, w, pre, dh)  # noqa: E731
    want = eager()
    d = [capi.DeviceArray.from_numpy(a) for a in (x, w, pre, dh)]
    out = [capi.DeviceArray(a.shape, dtype) for a in want]
    nb = lib.d8_matmul_gated_scratch_bytes(capi.dtype_id(dtype), 1, *size)
    ws = capi.DeviceArray((nb,), np.uint8)

    def call(stream):
        return lib.d8_matmul_gated_grad(capi.dtype_id(dtype), d[0].ptr, out[0].ptr, rows, inner, d[1].ptr, out[1].ptr, cols, 0, d[2].ptr, d[3].ptr, 3, ws.ptr, nb, stream)
    _replayed(call, out, want, eager)


def _rotary(cfg, dtype):
    """(arguments of the gradient call but for its outputs as a function of them, the eager results, a scratch size)"""
    from deep8_amd import capi, ops
    T, H, G, D, R, inter, norm, _ = cfg
    q, k, wq, wk, table, positions, gq, gk = rotary_inputs(cfg, dtype, 91)
    kw = dict(table=table, positions=positions, rotary=R, interleaved=inter, norm=norm)
    eager = lambda: ops.head_norm_rotary_grad(q, k, gq, gk, wq, wk, **kw)  # noqa: E731
    d = [None if a is None else capi.DeviceArray.from_numpy(a) for a in (q, wq, gq, k, wk, gk, positions, table)]
    p = [a and a.ptr for a in d]

    def call(out, dy, ws, nb, stream):
        dq, dwq, dk, dwk = (a and a.ptr for a in out)
        return capi.init().d8_head_norm_rotary_grad(capi.dtype_id(dtype), p[0], H * D, H, p[1], dy[0].ptr, H * D, dq, H * D, dwq, p[3], G * D, G, p[4], dy[1].ptr, G * D,
                                                    dk, G * D, dwk, T, D, int(norm), 1e-6, p[6], p[7], 50 if R else 0, R, int(inter), 3, ws.ptr, nb, stream)
    return call, eager, d, (gq, gk)


# 16-byte pieces in both layouts, several heads a group, no norm, the general kernel
PICKED = [c for c in ROTARY_CASES if c[:4] in ((5, 4, 2, 128), (700, 16, 8, 128), (9, 3, 3, 64), (33, 2, 1, 33), (33, 2, 1, 72))]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("cfg", PICKED)
def test_head_norm_rotary_grad(cfg, dtype):
    from deep8_amd import capi
    T, H, G, D, R, inter, norm, _ = cfg
    call, eager, d, grads = _rotary(cfg, dtype)
    dq, dk, dwq, dwk = eager()
    nb = capi.init().d8_head_norm_rotary_grad_scratch_bytes(capi.dtype_id(dtype), T, H, G, D)
    ws = capi.DeviceArray((nb,), np.uint8)
    out = [None if a is None else capi.DeviceArray(a.shape, dtype) for a in (dq, dwq, dk, dwk)]
    _replayed(lambda stream: call(out, (d[2], d[5]), ws, nb, stream), [a for a in out if a], [a for a in (dq, dwq, dk, dwk) if a is not None], eager)
    # over the gradients of the outputs
    over = [capi.DeviceArray.from_numpy(g) for g in grads]
    capi.check(call([over[0], out[1], over[1], out[3]], over, ws, nb, None))
    capi.sync()
    assert np.array_equal(over[0].numpy(), dq) and np.array_equal(over[1].numpy(), dk)
    if norm:
        assert np.array_equal(out[1].numpy(), dwq) and np.array_equal(out[3].numpy(), dwk)
