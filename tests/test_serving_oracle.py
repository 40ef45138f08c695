"""The 64-bit formulas that the norm of rows, the 8-bit products and the 8-bit cache are tested against: gradients against differences, the rest against
the attention formula and against what a rounding may do.

Differences as in test_layer_oracle.py: 1e-7 of the size."""
import numpy as np
import pytest

import layer_oracle as lo
import serving_oracle as so
from test_layer_oracle import _close, _differences
from util import rng


@pytest.mark.parametrize("epsilon", [1e-5, 0.5])
@pytest.mark.parametrize("weighted", [True, False])
def test_norm_of_rows(weighted, epsilon):
    r = rng(1)
    x, dy, w, b = r.standard_normal((4, 7)), r.standard_normal((4, 7)), r.standard_normal(7), r.standard_normal(7)
    if not weighted:
        w = None
    dx, dw, db = so.layer_norm_grad(x, dy, w, epsilon)
    _close(dx, _differences(lambda a: (so.layer_norm(a, w, b, epsilon)[0] * dy).sum(), x))
    if weighted:
        _close(dw, _differences(lambda a: (so.layer_norm(x, a, b, epsilon)[0] * dy).sum(), w))
    _close(db, _differences(lambda a: (so.layer_norm(x, w, a, epsilon)[0] * dy).sum(), b))
    u = so.layer_norm(x, None, None, 0.0)[1]
    assert np.abs(u.mean(1)).max() < 1e-15 and np.abs((u * u).mean(1) - 1).max() < 1e-14


def test_quantised_rows_are_half_a_step_off_at_most():
    x = rng(2).standard_normal((9, 50))
    x[3] = 0
    codes, scales = so.quantize(x)
    assert np.abs(codes).max() == 127 and not codes[3].any()
    # (the scale is the quotient by 127 rounded to 24 bits: 127 of it may miss the largest element by 127 parts in 2^24 of itself)
    assert (np.abs(codes * scales.astype(np.float64)[:, None] - x) <= scales[:, None] * (0.5 + 127 * 2.0 ** -24)).all()
    y, y_scales = so.quantize(rng(3).standard_normal((5, 50)))
    want = (codes * scales.astype(np.float64)[:, None]) @ (y * y_scales.astype(np.float64)[:, None]).T
    assert np.abs(so.matmul_int8(codes, scales, y, y_scales) - want).max() <= 1e-12


@pytest.mark.parametrize("steps", [[70, 60], [1] * 130, [64, 1, 65]])
def test_cache_holds_its_tokens_to_half_a_step(steps):
    """tokens as they come, pages in any order: what is read back is within half a step of the page's scale, and half a step of each smaller one that the
    page went through (those are powers of two: together less than one step)"""
    r, G, D, table = rng(4), 2, 6, np.array([[4, 0, 2]], np.int32)
    cache, n = so.Cache(5, G, D), sum(steps)
    k, v = r.standard_normal((n, G, D)), 10 * r.standard_normal((n, G, D))
    at = 0
    for step in steps:
        cache.append(k[at:at + step], v[at:at + step], [0, step], [at + step], table)
        at += step
    back = cache.read(n, [0, n], [n], table, (k, v))
    for name, x, y in (("k", k, back[0]), ("v", v, back[1])):
        for t in range(n):
            scale = cache.scales[name][table[0, t // 64]]
            assert (np.abs(x[t] - y[t]) <= scale[:, None]).all()
            assert (np.log2(scale) % 1 == 0).all()
    if len(steps) == 2:  # a page that is written at once: half a step
        assert (np.abs(k[:64] - back[0][:64]) <= cache.scales["k"][4][:, None] / 2).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("new,lengths", [([3, 2], [70, 2]), ([1, 1], [128, 65]), ([0, 4], [0, 9])])
def test_attention_over_pages_is_attention_over_their_values(new, lengths, causal):
    r, H, G, D = rng(5), 4, 2, 3
    table = np.array([[3, 1], [0, 2]], np.int32)
    kv, vv = r.standard_normal((4, G, 64, D)), r.standard_normal((4, G, 64, D))
    starts = np.concatenate([[0], np.cumsum(new)])
    q = r.standard_normal((starts[-1], H, D))
    flat = [np.concatenate([np.concatenate([a[p].transpose(1, 0, 2) for p in table[s]])[:n] for s, n in enumerate(lengths)]) for a in (kv, vv)]
    want = lo.attention(q, *flat, starts, np.concatenate([[0], np.cumsum(lengths)]), 0.7, causal)
    got = so.attention_cache(q, kv, vv, starts, lengths, table, 4, 0.7, causal)
    for g, w in zip(got, want):
        assert np.abs(g - w).max() <= 1e-12
