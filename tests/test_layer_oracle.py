"""The 64-bit formulas that the layer operators are tested against, their gradients checked against differences.

A central difference over h = 1e-5 of a function with third derivatives of order 1 is off by h^2 = 1e-10 and by the rounding of the two
values, 1e-16 times their size (up to some hundreds here) over h: 1e-9.  A hundred times that is allowed."""
import numpy as np
import pytest

import layer_oracle as lo
from util import rng

H = 1e-5
TOL = 1e-7


def _differences(f, x):
    """gradient of the number f(x) by differences"""
    g = np.zeros_like(x)
    for i in np.ndindex(x.shape):
        up, down = x.copy(), x.copy()
        up[i] += H
        down[i] -= H
        g[i] = (f(up) - f(down)) / (2 * H)
    return g


def _close(got, want):
    assert np.abs(got - want).max() <= TOL * max(1.0, np.abs(want).max())


@pytest.mark.parametrize("rotary,interleaved,norm", [(6, False, True), (4, True, True), (0, False, True), (6, True, False)])
def test_norm_rotary(rotary, interleaved, norm):
    r = rng(1)
    x, dy, w = r.standard_normal((3, 2, 6)), r.standard_normal((3, 2, 6)), r.standard_normal(6) if norm else None
    t = lo.table(9, rotary) if rotary else None
    args = t, np.array([5, 0, 8]), rotary, interleaved, norm
    dx, dw = lo.norm_rotary_grad(x, w, dy, *args)
    _close(dx, _differences(lambda a: (lo.norm_rotary(a, w, *args) * dy).sum(), x))
    if norm:
        _close(dw, _differences(lambda a: (lo.norm_rotary(x, a, *args) * dy).sum(), w))


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", [([3, 2], [3, 4]), ([4], [2]), ([0, 2], [3, 0])])
def test_attention(causal, nq, nk):
    r = rng(2)
    qs, ks = np.concatenate([[0], np.cumsum(nq)]), np.concatenate([[0], np.cumsum(nk)])
    q, k, v = r.standard_normal((qs[-1], 4, 3)), r.standard_normal((ks[-1], 2, 3)), r.standard_normal((ks[-1], 2, 3))
    do = r.standard_normal(q.shape)
    dq, dk, dv = lo.attention(q, k, v, qs, ks, 0.7, causal, do)
    _close(dq, _differences(lambda a: (lo.attention(a, k, v, qs, ks, 0.7, causal)[0] * do).sum(), q))
    _close(dk, _differences(lambda a: (lo.attention(q, a, v, qs, ks, 0.7, causal)[0] * do).sum(), k))
    _close(dv, _differences(lambda a: (lo.attention(q, k, a, qs, ks, 0.7, causal)[0] * do).sum(), v))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_gated(act):
    r = rng(3)
    x, w, dh = r.standard_normal((3, 4)), r.standard_normal((4, 6)), r.standard_normal((3, 3))
    dx, dw = lo.gated_grad(x, w, lo.gated(x, w, act)[1], dh, act)
    _close(dx, _differences(lambda a: (lo.gated(a, w, act)[0] * dh).sum(), x))
    _close(dw, _differences(lambda a: (lo.gated(x, a, act)[0] * dh).sum(), w))
