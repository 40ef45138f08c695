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
