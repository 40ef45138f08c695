"""d8_attention_cache at the ends of what scores and values can be."""
import numpy as np
import pytest

from util import f

PAGE = 64


def _cache(k, v, k_scales, v_scales):
    """codes [page][token][dim] of one head, scales [page]"""
    from deep8_amd import ops
    cache = ops.PagedCache(len(k), 1, k.shape[2])
    cache.k_codes.copy_from(np.ascontiguousarray(k[:, None].astype(np.int8)))
    cache.v_codes.copy_from(np.ascontiguousarray(v[:, None].swapaxes(2, 3).astype(np.int8)))
    cache.k_scales.copy_from(np.asarray(k_scales, np.float32)[:, None])
    cache.v_scales.copy_from(np.asarray(v_scales, np.float32)[:, None])
    return cache


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [1, 7])
@pytest.mark.parametrize("order", [[0, 1, 2], [2, 1, 0], [1, 0, 2]])
def test_scores_of_any_size(order, n, dtype):
    """scores of 2^12 to 2^41, gaps of 2^6 and more: the result is the values of the key that has the largest, exactly (its weight is a power of two, and so are
    the pages' scales); lse is its score, of seven factors and products rounded to 24 bits each"""
    r = np.random.default_rng(n)
    k, v = np.zeros((3, PAGE, 16), int), r.integers(-127, 128, (3, PAGE, 16))
    k[:, :, 0] = np.arange(PAGE)
    cache = _cache(k, v, [1, 0.5, 0.25], [2.0 ** -6, 2.0 ** -3, 1])
    e = np.repeat(np.arange(16), n)
    q = np.zeros((len(e), 1, 16), dtype)
    q[:, 0, 0] = 2.0 ** e
    for scale in (2.0 ** 6, 2.0 ** 20):
        got, lse = cache.attention(q, [0, len(e)], [3 * PAGE], [order], scale, False)
        assert np.array_equal(f(got)[:, 0], np.broadcast_to((v[0, -1] * 2.0 ** -6).astype(np.float32), (len(e), 16)))
        score = 2.0 ** e * 63 * scale
        assert (np.abs(lse[0] - score) <= 8 * 2.0 ** -24 * score).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("keys", [1, 64, 700])
@pytest.mark.parametrize("top", [65504, 65472, 61000, 40000])
def test_values_next_to_the_largest_half(top, keys, n):
    """codes of the largest halves may stand for more than a half holds (65504 is 64 steps of 1024); the cache is read as 65504 there, and so is a mean of such
    values, which is off by half a step of 1024, of the sums' fp32 and of its own rounding, 2^-11 (weights: all alike)"""
    from deep8_amd import ops
    pages = -(-keys // PAGE)
    cache, table = ops.PagedCache(pages, 1, 32), np.arange(pages, dtype=np.int32)[None]
    v = np.zeros((keys, 1, 32), np.float16)
    v[:] = np.array([top, -top, top / 2, 1] * 8)
    cache.append(np.ones_like(v), v, [0, keys], [keys], table)
    back = cache.read(keys, [0, keys], [keys], table, np.float16)[1]
    got, lse = cache.attention(np.ones((n, 1, 32), np.float16), [0, n], [keys], table, 0.125, False)
    got = f(got)[:, 0].astype(np.float64)
    assert np.isfinite(got).all()
    assert (np.abs(got - f(back)[0, 0]) <= 2.0 ** -10 * np.abs(f(back)[0, 0])).all()
    assert (np.abs(got - f(v)[0, 0]) <= 512 + 2.0 ** -10 * np.abs(f(v)[0, 0])).all()
    assert (np.abs(lse - (4 + np.log(keys))) <= 1e-5 * 12).all()
