"""d8_attention_cache where sequences are long: weights far below the row's largest, and runs of many pages.

A table may name a full page any number of times, so a long sequence takes a few pages' memory."""
import numpy as np
import pytest

import serving_oracle as so
from util import f

PAGE = 64


def _pages(codes, scales):
    """a cache of these codes [k or v][page][head][token][dim] and scales [k or v][page][head], and its values in 64 bits"""
    from deep8_amd import ops
    pages, heads, _, dim = codes[0].shape
    cache, values = ops.PagedCache(pages, heads, dim), []
    for name, x, s in zip("kv", codes, scales):
        x = np.pad(x.astype(np.int8), ((0, 0), (0, 0), (0, 0), (0, cache.pitch - dim)))
        getattr(cache, name + "_codes").copy_from(x if name == "k" else np.ascontiguousarray(x.swapaxes(2, 3)))
        getattr(cache, name + "_scales").copy_from(s.astype(np.float32))
        values.append(x[..., :dim].astype(np.float64) * s.astype(np.float32).astype(np.float64)[..., None, None])
    return cache, values


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [1, 100])
@pytest.mark.parametrize("below", [24.55, 25.05, 30.0])
def test_many_small_weights_beside_a_large_one(below, n, dtype):
    """the first key, whose values are zero, takes nearly all the weight; the result is what 131071 others, 2^-below of it each, add up to.  (256 heads, all alike:
    a run is half the sequence, which has met the large weight before the small ones.)

    A weight as half is off by 2^-11 of itself, all alike here (single: two halves), or, where it is small, by 2^-25 of 2^14 times itself: 2^-39 of the row's
    largest, which N of them add up.  The result is rounded once more; scores of some 20 times log2 e in fp32 make the weights 1e-5 uncertain.  And both sums go
    through N / 64 pages one after the other in fp32, off by 2^-24 of themselves each time, and always to the same side where all terms are alike: 2048 2^-23."""
    N, H = 131072, 256
    r = np.random.default_rng(int(below))
    k, v = np.full((2, 1, PAGE, 16), -28), r.integers(1, 128, (2, 1, PAGE, 16))
    k[0, 0, 0], v[0, 0, 0] = 100, 0
    cache, (kv, vv) = _pages([a.repeat(H, 1) for a in (k, v)], (np.full((2, H), 2.0 ** -5), np.full((2, H), 2.0 ** -6)))
    table = np.ones((1, N // PAGE), np.int32)
    table[0, 0] = 0
    q = np.zeros((n, H, 16), dtype)
    q[:, :, 0] = 1
    scale = below * np.log(2) / 4  # the two keys' scores: 128 codes of 2^-5 apart
    want, lse = so.attention_cache(q[:1, :1], kv[:, :1], vv[:, :1], [0, 1], [N], table, 2, scale, False)
    got, got_lse = cache.attention(q, [0, n], [N], table, scale, False)
    near = 2.0 ** -10 if dtype == np.float16 else 2.0 ** -20
    bound = (near + 1e-5 + N / PAGE * 2.0 ** -23) * want[0, 0] + N * 2.0 ** -39 * 2 + (2.0 ** -25 if dtype == np.float16 else 0)
    over = np.abs(f(got).astype(np.float64) - want[0, 0]) / bound
    assert over.max() <= 1
    assert (np.abs(got_lse - lse[0, 0]) <= 1e-5 * abs(lse[0, 0])).all()
