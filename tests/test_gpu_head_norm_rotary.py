"""d8_head_norm_rotary, its gradient and d8_rotary_table against the formulas in 64 bits.

Tolerances (relative Frobenius, and per token against that token's norm and the mean one).  Float16: values and gradients are
rounded once, at most 2^-11 = 4.9e-4, or 2^-25 where they are subnormal (the gradient of a head of one element is of
the size of epsilon).  Float32: a few dozen roundings of 2^-24 = 6e-8 in the longest chain of one element: 2e-6; a weight's gradient
is a sum over tokens and heads whose terms cancel, sqrt(rows) times smaller than the sum of their sizes: 1e-5.  The
table holds fp32 roundings of values of at most 1: 6e-8."""
import numpy as np
import pytest

import layer_oracle as lo
from util import f, rel_fro, rng

pytestmark = pytest.mark.gpu
TOL = {np.float16: 4.9e-4, np.float32: 2e-6}
WEIGHT_TOL = {np.float16: 5e-4, np.float32: 1e-5}

CASES = [
    # tokens, q heads, k heads, dim, rotary, interleaved, norm, pad
    (5, 4, 2, 128, 128, False, True, 0),    # 16-byte pieces, half layout
    (5, 4, 2, 128, 128, True, True, 8),     # neighbours, rows apart
    (67, 12, 4, 96, 64, True, True, 16),    # part of the head
    (300, 5, 1, 80, 32, False, True, 0),    # a remainder of an odd number of pieces
    (9, 3, 3, 64, 0, False, True, 0),       # norm alone
    (9, 3, 3, 64, 64, False, False, 0),     # rotation alone
    (33, 2, 1, 33, 10, False, True, 3),     # the general kernel: odd heads, odd rows
    (33, 2, 1, 72, 12, False, True, 0),     # ... pairs that straddle pieces
    (4, 1, 1, 7, 6, True, True, 1),
    (3, 2, 0, 64, 64, False, True, 0),      # queries alone
    (1, 0, 3, 1, 0, False, True, 0),        # keys alone, heads of one element
    (2, 1, 2, 512, 256, False, True, 0),    # heads as wide as a wave
    (2, 1, 1, 2048, 2048, True, True, 0),
    (700, 16, 8, 128, 128, False, True, 0), # several heads a group
    (0, 2, 1, 64, 64, False, True, 0),      # no token
]


def _near(got, want, tol):
    half = got.dtype == np.float16
    got, want = f(got).astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    if not want.size:
        return
    assert np.linalg.norm(got - want) <= tol * np.linalg.norm(want) + (2.0 ** -25 * np.sqrt((np.abs(want) < 2.0 ** -14).sum()) if half else 0)
    if half and np.abs(want).max() < 2.0 ** -14:
        return
    e, n = np.linalg.norm((got - want).reshape(len(want), -1), axis=1), np.linalg.norm(want.reshape(len(want), -1), axis=1)
    assert (e <= 4 * tol * (n + n.mean())).all()


def _inputs(cfg, dtype, seed):
    T, H, G, D, R, inter, norm, pad = cfg
    r = rng(seed)
    c = lambda *s: r.standard_normal(s).astype(dtype)  # noqa: E731
    q, k = c(T, H, D) * dtype(2), c(T, G, D)
    wq, wk = (c(D), c(D)) if norm else (None, None)
    table = lo.table(50, R).astype(np.float32) if R else None
    positions = r.integers(-3, 60, T).astype(np.int32)  # some outside the table: they count as its ends
    return q, k, wq, wk, table, positions, c(T, H, D), c(T, G, D)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("cfg", CASES)
def test_forward_and_gradient(cfg, dtype):
    from deep8_amd import ops
    T, H, G, D, R, inter, norm, pad = cfg
    q, k, wq, wk, table, positions, gq, gk = _inputs(cfg, dtype, sum(cfg))
    kw = dict(table=table, positions=positions, rotary=R, interleaved=inter, norm=norm)
    args = table, positions, R, inter, norm
    want = lo.norm_rotary(q, wq, *args), lo.norm_rotary(k, wk, *args)
    got = ops.head_norm_rotary(q, k, wq, wk, pad=pad, **kw)
    for g, w in zip(got, want):
        _near(g, w, TOL[dtype])
    again = ops.head_norm_rotary(q, k, wq, wk, pad=pad, in_place=True, **kw)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))
    back = lo.norm_rotary_grad(q, wq, gq, *args), lo.norm_rotary_grad(k, wk, gk, *args)
    dq, dk, dwq, dwk = ops.head_norm_rotary_grad(q, k, gq, gk, wq, wk, pad=pad, **kw)
    _near(dq, back[0][0], TOL[dtype])
    _near(dk, back[1][0], TOL[dtype])
    if norm:
        scale = np.linalg.norm(f(gq)) + np.linalg.norm(f(gk)) + 1e-30
        for g, w in ((dwq, back[0][1]), (dwk, back[1][1])):
            assert np.linalg.norm(f(g) - w) <= WEIGHT_TOL[dtype] * max(np.linalg.norm(w), scale)
    # added to what is there
    old = [np.ones_like(a) if a is not None else None for a in (dq, dk, dwq, dwk)]
    summed = ops.head_norm_rotary_grad(q, k, gq, gk, wq, wk, pad=pad, into=old, **kw)
    _near(summed[0], back[0][0] + 1, 2 * TOL[dtype])
    if norm:
        assert np.abs(f(summed[2]) - f(dwq) - 1).max(initial=0) <= 4 * TOL[dtype] * (1 + np.abs(f(dwq)).max(initial=0))


def test_positions_by_row_and_default_weights():
    from deep8_amd import ops
    q, k, _, _, table, _, gq, gk = _inputs((40, 2, 1, 64, 64, False, True, 0), np.float32, 3)
    args = table, None, 64, False, True
    got = ops.head_norm_rotary(q, k, table=table, rotary=64)
    _near(got[0], lo.norm_rotary(q, None, *args), TOL[np.float32])
    dq, dk, dwq, dwk = ops.head_norm_rotary_grad(q, k, gq, gk, table=table, rotary=64)
    _near(dk, lo.norm_rotary_grad(k, None, gk, *args)[0], TOL[np.float32])
    assert dwq is None and dwk is None


def test_rows_of_zeros_infinities_and_nan():
    """a head of zeros stays one; a head that holds what is no number does not touch its neighbours"""
    from deep8_amd import ops
    q, k, wq, wk, table, positions, gq, gk = _inputs((6, 2, 1, 128, 128, False, True, 0), np.float16, 4)
    q[1], q[2, 0, 3], q[3, 1, 7] = 0, np.inf, np.nan
    kw = dict(table=table, positions=positions, rotary=128)
    got, clean = ops.head_norm_rotary(q, k, wq, wk, **kw)[0], lo.norm_rotary(np.nan_to_num(f(q), posinf=0), wq, table, positions, 128, False, True)
    assert (got[1] == 0).all() and np.isnan(got[3, 1]).all() and np.isnan(got[2, 0]).any()
    for t, h in ((0, 0), (2, 1), (3, 0), (4, 0), (5, 1)):
        assert rel_fro(f(got[t, h]), clean[t, h]) <= TOL[np.float16]


@pytest.mark.parametrize("kw", [{}, {"factor": 4.0}, {"factor": 8.0, "keep_below": 40.0, "slow_above": 4000.0}, {"base": 500000.0}])
def test_table(kw):
    from deep8_amd import ops
    got = ops.rotary_table(5000, 64, **kw)
    assert np.abs(got - lo.table(5000, 64, **kw)).max() <= 6.1e-8
    assert np.abs(ops.rotary_table(70000, 6)[-1] - lo.table(70000, 6)[-1]).max() <= 6.1e-8


def test_refusals():
    from deep8_amd import capi, ops
    x = np.zeros((2, 1, 8), np.float32)
    t = np.zeros((4, 4, 2), np.float32)
    for kw in (dict(rotary=3, table=t), dict(rotary=10, table=t), dict(rotary=8), dict(rotary=-2, table=t)):
        with pytest.raises(capi.Deep8HipError):
            ops.head_norm_rotary(x, x, **kw)
    with pytest.raises(capi.Deep8HipError):  # a weight, but no norm
        ops.head_norm_rotary(x, x, q_weight=np.ones(8), norm=False)
    with pytest.raises(capi.Deep8HipError):
        ops.head_norm_rotary(x.astype(np.float64), x.astype(np.float64))
    with pytest.raises(capi.Deep8HipError):
        ops.head_norm_rotary(np.zeros((1, 1, 2049), np.float32), np.zeros((1, 1, 2049), np.float32))
    with pytest.raises(capi.Deep8HipError):
        ops.rotary_table(4, 5)
    with pytest.raises(capi.Deep8HipError):
        ops.rotary_table(4, 4, keep_below=8.0, slow_above=4.0)
    lib = capi.init()
    d = capi.DeviceArray((2, 8))
    assert lib.d8_head_norm_rotary(capi.FLOAT32, d.ptr, 7, 1, None, d.ptr, 8, None, 0, 0, None, None, 0, 2, 8, 1, 1e-6, None, None, 0, 0, 0, None) == 10001
    assert lib.d8_head_norm_rotary(capi.FLOAT32, None, 8, 1, None, d.ptr, 8, None, 0, 0, None, None, 0, 2, 8, 1, 1e-6, None, None, 0, 0, 0, None) == 10001
    assert b"null" in lib.d8_last_error()
