"""d8_attention and d8_attention_grad against the formulas in 64 bits.

Tolerances (relative Frobenius, and per row against that row's norm and the mean one): the framework's, 1e-5 in Float32 and 2e-3 in
Float16.  What goes in: Float32, sums of at most a thousand terms, each rounded to 2^-24, and scores of up to 20 whose
rounding the exponential turns into a relative error of 20 * 2^-24 = 1.2e-6.  Float16, roundings to half of 2^-11 at most
in the probabilities, the result, and on the way back the score's gradient and the forward result behind delta: four of them, 2e-3."""
import numpy as np
import pytest

import layer_oracle as lo
from util import FP16_TOL, FP32_TOL, f, rel_fro, rng

pytestmark = pytest.mark.gpu
TOL = {np.float16: FP16_TOL, np.float32: FP32_TOL}

CASES = [
    # queries, keys of each sequence, heads, kv heads, dim, causal, pad
    ([5], [5], 1, 1, 8, True, 0),
    ([1], [1], 2, 1, 64, True, 0),
    ([130, 7, 64], [130, 7, 64], 4, 2, 64, True, 0),       # several tiles, one, none more
    ([33, 1, 0, 31, 200], [33, 1, 0, 31, 200], 6, 2, 80, True, 16),
    ([40, 9], [100, 70], 3, 3, 128, True, 0),              # a prompt's next part
    ([1, 1, 1, 1], [300, 1, 64, 129], 8, 2, 128, True, 0), # decoding
    ([1, 1], [900, 1000], 5, 1, 96, True, 8),
    ([4, 2], [2, 0], 2, 1, 32, True, 0),                   # queries that see nothing
    ([0, 3], [5, 0], 2, 2, 64, False, 0),                  # keys without queries, queries without keys
    ([70, 90], [50, 200], 4, 1, 64, False, 0),             # every key, of lengths of its own
    ([50], [50], 3, 1, 33, True, 3),                       # rows that start anywhere
    ([37], [64], 2, 2, 7, False, 1),
    ([20, 70], [20, 70], 2, 1, 256, True, 0),              # the widest heads
    ([20, 70], [20, 70], 2, 1, 200, False, 1),
    ([128, 256], [128, 256], 4, 4, 128, True, 0),          # whole tiles
    ([257], [511], 16, 2, 64, True, 0),
    ([1] * 70, [3] * 70, 2, 2, 32, True, 0),               # more sequences than lanes of a wave
]


def _near(got, want, tol):
    got, want = f(got).astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    if not want.size:
        return
    assert rel_fro(got, want) <= tol
    e, n = np.linalg.norm((got - want).reshape(len(want), -1), axis=1), np.linalg.norm(want.reshape(len(want), -1), axis=1)
    assert (e <= 4 * tol * (n + n.mean())).all()


def _starts(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def _inputs(nq, nk, H, G, D, dtype, seed):
    r = rng(seed)
    c = lambda *s: r.standard_normal(s).astype(dtype)  # noqa: E731
    return c(sum(nq), H, D), c(sum(nk), G, D), c(sum(nk), G, D), c(sum(nq), H, D)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("cfg", CASES)
def test_forward_and_gradient(cfg, dtype):
    from deep8_amd import ops
    nq, nk, H, G, D, causal, pad = cfg
    q, k, v, do = _inputs(nq, nk, H, G, D, dtype, sum(nq) + 7 * D)
    qs, ks, scale = _starts(nq), _starts(nk), D ** -0.5
    want, lse = lo.attention(q, k, v, qs, ks, scale, causal)
    got, got_lse = ops.attention(q, k, v, qs, ks, scale, causal, pad=pad)
    _near(got, want, TOL[dtype])
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got_lse), empty) and (f(got)[empty.T] == 0).all()
    assert np.abs(got_lse[~empty] - lse[~empty]).max(initial=0) <= 1e-5 * max(1, np.abs(lse[~empty]).max(initial=0))
    grads = lo.attention(q, k, v, qs, ks, scale, causal, do)
    back = ops.attention_grad(q, k, v, got, got_lse, do, qs, ks, scale, causal, pad=pad)
    norm = np.linalg.norm(f(do))
    for g, w in zip(back, grads):
        if np.linalg.norm(w) > 1e-3 * norm:
            _near(g, w, TOL[dtype])
        else:  # gradients that cancel (a query with one key has none): against the size of their terms
            assert np.linalg.norm(f(g) - w) <= TOL[dtype] * norm
    assert (f(back[0])[empty.T] == 0).all()
    again = ops.attention_grad(q, k, v, got, got_lse, do, qs, ks, scale, causal, pad=pad)
    assert all(np.array_equal(a, b) for a, b in zip(back, again))
    old = [np.ones_like(a) for a in back]
    summed = ops.attention_grad(q, k, v, got, got_lse, do, qs, ks, scale, causal, pad=pad, into=old)
    for s, w in zip(summed, grads):
        _near(s, w + 1, 2 * TOL[dtype])


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("dim,H,G,causal", [(32, 16, 16, True), (64, 16, 16, True), (80, 24, 12, True), (128, 16, 16, True), (128, 15, 15, False), (256, 16, 16, True), (200, 16, 8, False)])
def test_many_rows(dtype, dim, H, G, causal):
    """enough rows for workgroups of 128 of them; lengths that end inside tiles of rows and of keys, queries fewer and more than keys"""
    from deep8_amd import ops
    r = rng(dim + H)
    nq = list(r.integers(150, 390, 15)) + [1, 300]
    nk = [int(max(0, n + r.integers(-70, 130))) for n in nq]
    q, k, v, do = _inputs(nq, nk, H, G, dim, dtype, dim)
    qs, ks, scale = _starts(nq), _starts(nk), -(dim ** -0.5)
    want, lse = lo.attention(q, k, v, qs, ks, scale, causal)
    got, got_lse = ops.attention(q, k, v, qs, ks, scale, causal, pad=8)
    _near(got, want, TOL[dtype])
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got_lse), empty) and np.abs(got_lse - lse)[~empty].max() <= 1e-5 * np.abs(lse[~empty]).max()
    grads = lo.attention(q, k, v, qs, ks, scale, causal, do)
    back = ops.attention_grad(q, k, v, got, got_lse, do, qs, ks, scale, causal, pad=8)
    for g, w in zip(back, grads):
        _near(g, w, TOL[dtype])


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_long_cache(dtype):
    """one query against tens of thousands of keys, the largest score far from the first"""
    from deep8_amd import ops
    nq, nk = [1, 3, 1], [20001, 9000, 33]
    q, k, v, _ = _inputs(nq, nk, 8, 2, 64, dtype, 5)
    k[15000] = 4 * q[0, :2]
    qs, ks = _starts(nq), _starts(nk)
    want, lse = lo.attention(q, k, v, qs, ks, 0.125, True)
    got, got_lse = ops.attention(q, k, v, qs, ks, 0.125, True)
    _near(got, want, TOL[dtype])
    assert np.abs(got_lse - lse).max() <= 2e-5 * np.abs(lse).max()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_large_and_equal_scores(dtype):
    """scores of some thousands (the exponential of a score itself would overflow), and all scores equal"""
    from deep8_amd import ops
    q, k, v, do = _inputs([40], [40], 2, 2, 64, np.float16, 6)
    q, k, v, do = (a.astype(dtype) for a in (q, k, v, do))
    s = _starts([40])
    want, _ = lo.attention(q, k, v, s, s, 30.0, True)
    got, lse = ops.attention(q, k, v, s, s, 30.0, True)
    _near(got, want, 20 * TOL[dtype])  # scores of about 1000: their rounding, 2^-24 of it, goes into the exponent
    want, _ = lo.attention(q, k, v, s, s, 0.0, True)
    got, lse = ops.attention(q, k, v, s, s, 0.0, True)
    _near(got, want, TOL[dtype])
    assert np.allclose(lse, np.log(np.arange(1, 41)), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_small_probabilities_and_gradients(dtype):
    """probabilities of 2^-12 and output gradients of 2^-9: half's subnormals must not swallow them on the way back"""
    from deep8_amd import ops
    q, k, v, do = _inputs([512], [4096], 1, 1, 64, dtype, 8)
    do = (f(do) / 512).astype(dtype)
    k = (f(k) / 8).astype(dtype)
    qs, ks = _starts([512]), _starts([4096])
    o, lse = ops.attention(q, k, v, qs, ks, 0.125, False)
    back = ops.attention_grad(q, k, v, o, lse, do, qs, ks, 0.125, False)
    want = lo.attention(q, k, v, qs, ks, 0.125, False, do)
    for g, w in zip(back, want):
        if dtype == np.float32:
            _near(g, w, FP32_TOL)
        else:  # the results themselves are subnormal halves: 2^-25 of rounding each
            assert np.linalg.norm(f(g) - w) <= FP16_TOL * np.linalg.norm(w) + 2.0 ** -25 * np.sqrt(w.size)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_what_lies_outside_a_sequence_does_not_reach_it(dtype):
    """NaN and infinities in the other sequences, in rows of no sequence and in keys that no query of the tile sees"""
    from deep8_amd import ops
    nq = [20, 45, 9, 300]
    q, k, v, do = _inputs(nq, nq, 4, 2, 64, dtype, 9)
    s = _starts(nq)
    clean = q.copy(), k.copy(), v.copy(), do.copy()
    for a, bad in ((q, np.nan), (k, np.inf), (v, np.nan), (do, np.nan)):
        a[s[1]:s[2]] = bad
    k[-1], v[-1] = np.nan, np.nan  # the last key of the last sequence: only its last query sees it
    starts = s[[0, 1, 2, 3, 4]].copy()
    want = lo.attention(*clean[:3], s, s, 0.125, True)[0]
    got, lse = ops.attention(q, k, v, starts, starts, 0.125, True)
    for part in (slice(0, 20), slice(s[2], s[3]), slice(s[3], s[3] + 128)):
        _near(got[part], want[part], TOL[dtype])
    assert np.isnan(f(got[s[1]:s[2]])).all()
    # rows before, between and after the sequences stay as they are
    inner = np.array([25, 60, 70], np.int32)
    left = np.full_like(q, 7)
    got, lse = ops.attention(*clean[:3], inner, inner, 0.125, True, o=left)
    want, _ = lo.attention(*clean[:3], inner, inner, 0.125, True)
    assert (got[:25] == 7).all() and (got[70:] == 7).all() and np.isnan(lse[:, :25]).all()
    _near(got[25:70], want[25:70], TOL[dtype])


def test_starts_beyond_the_tensors_are_cut():
    from deep8_amd import ops
    q, k, v, do = _inputs([50], [50], 2, 1, 64, np.float32, 10)
    wild = np.array([-5, 30, 20, 1 << 30], np.int32)
    got, lse = ops.attention(q, k, v, wild, wild, 0.125, True)
    want, _ = lo.attention(q, k, v, [0, 30], [0, 30], 0.125, True)
    _near(got[:20], want[:20], FP32_TOL)
    ops.attention_grad(q, k, v, got, np.nan_to_num(lse), do, wild, wild, 0.125, True)


def test_stream_and_graph():
    """a captured call replays to the same bits as the eager one, on a stream of its own"""
    import ctypes
    from deep8_amd import capi, ops
    lib = capi.init()
    q, k, v, _ = _inputs([1, 1, 1], [700, 2000, 5], 8, 2, 128, np.float16, 11)
    qs, ks = _starts([1, 1, 1]), _starts([700, 2000, 5])
    want, want_lse = ops.attention(q, k, v, qs, ks, 0.1, True)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    capi.check(lib.d8_stream_create(ctypes.byref(stream)))
    d = [capi.DeviceArray.from_numpy(a) for a in (q, k, v, np.zeros_like(q), np.zeros((8, 3), np.float32), qs, ks)]
    n = 3, 3, 2705, 8, 2, 128
    nb = lib.d8_attention_scratch_bytes(capi.FLOAT16, 0, *n, 1)
    ws = capi.DeviceArray((max(nb, 16),), np.uint8)
    capi.check(lib.d8_graph_begin(stream))
    rc = lib.d8_attention(capi.FLOAT16, d[0].ptr, 1024, d[1].ptr, 256, d[2].ptr, 256, d[3].ptr, 1024, d[4].ptr, d[5].ptr, d[6].ptr, *n, 0.1, 1, ws.ptr, nb, stream)
    capi.check(lib.d8_graph_end(stream, ctypes.byref(graph)))
    capi.check(rc)
    for _ in range(3):
        d[3].copy_from(np.zeros_like(q))
        d[4].copy_from(np.zeros((8, 3), np.float32))
        capi.check(lib.d8_graph_launch(graph, stream))
        capi.sync(stream)
        assert np.array_equal(d[3].numpy(), want) and np.array_equal(d[4].numpy(), want_lse)
    capi.check(lib.d8_graph_destroy(graph))
    capi.check(lib.d8_stream_destroy(stream))


def test_refusals():
    from deep8_amd import capi, ops
    q = np.zeros((2, 4, 8), np.float32)
    s = np.array([0, 2], np.int32)
    bad = np.zeros((2, 3, 8), np.float32)
    with pytest.raises(capi.Deep8HipError):
        ops.attention(q, bad, bad, s, s, 1.0)  # 4 heads on 3
    with pytest.raises(capi.Deep8HipError):
        ops.attention(q, q, q, s, s, float("nan"))
    with pytest.raises(capi.Deep8HipError):
        ops.attention(*(a.astype(np.float64) for a in (q, q, q)), s, s, 1.0)
    wide = np.zeros((2, 1, 257), np.float16)
    with pytest.raises(capi.Deep8HipError):
        ops.attention(wide, wide, wide, s, s, 1.0)
    lib = capi.init()
    d, i = capi.DeviceArray((2, 32)), capi.DeviceArray.from_numpy(s)
    call = lambda **k: lib.d8_attention(capi.FLOAT32, k.get("q", d.ptr), k.get("ldq", 32), d.ptr, 32, d.ptr, 32, d.ptr, 32, None, k.get("s", i.ptr), i.ptr,  # noqa: E731
                                        k.get("n", 1), 2, 2, 4, 4, 8, 1.0, 1, None, 0, None)
    assert call() == 0
    assert call(q=None) == 10001 and call(s=None) == 10001 and call(ldq=31) == 10001 and call(n=-1) == 10001
    assert lib.d8_attention_grad(capi.FLOAT32, d.ptr, 32, d.ptr, 32, d.ptr, 32, d.ptr, 32, d.ptr, d.ptr, 32, d.ptr, 32, d.ptr, 32, d.ptr, 32, i.ptr, i.ptr, 1, 2, 2, 4, 4, 8,
                                 1.0, 1, 7, None, 0, None) == 10001
    assert b"scratch" in lib.d8_last_error()
