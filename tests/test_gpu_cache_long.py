"""d8_attention_cache where sequences are long: weights far below the row's largest, and runs of many pages.

A table may name a full page any number of times, so a long sequence takes a few pages' memory."""
import numpy as np
import pytest

import serving_oracle as so
from util import FP16_TOL, FP32_TOL, f, rel_fro

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


# queries and pages of each sequence, query heads a key head, key heads, dim, causal; the pages that the longest run of a call has in one sequence, at least:
# few rows (a wave has every fourth of them, 64 at a time), then many (all waves go through them together, 64 at a time)
RUNS = [([1], [40], 1, 256, 64, True, 20),
        ([1], [37], 3, 256, 128, True, 19),
        ([1], [600], 1, 256, 64, True, 300),
        ([1, 2, 1], [520, 3, 130], 2, 256, 16, True, 300),
        ([5], [300], 2, 128, 128, False, 75),
        ([1, 1], [30, 290], 1, 256, 200, True, 160),
        ([9], [64], 1, 128, 256, True, 32),
        ([130], [150], 1, 128, 64, True, 75),
        ([100], [140], 1, 256, 128, False, 70),
        ([40, 70], [90, 160], 3, 256, 48, True, 75)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rising", ["late", "early", "anywhere"])
@pytest.mark.parametrize("nq,np_,group,G,D,causal,least", RUNS)
def test_runs_of_many_pages(nq, np_, group, G, D, causal, least, rising, dtype):
    """many key heads leave few runs, so that each goes through many pages: scores that grow along a sequence, sums that are scaled down once and again, and the
    other way round.  Tolerances as test_gpu_cache.py's: 2e-3 and 1e-5 of the row's and the rows' mean size"""
    from deep8_amd import capi
    H, n, width = G * group, sum(nq), max(np_) + 1
    lib, dt = capi.init(), capi.dtype_id(dtype)
    many = D <= 128 and n * group // len(nq) >= (33 if dtype == np.float16 else 96)
    tile = 128 if many else 16
    # how long the runs are, from the scratch that the call asks for (a slot for each tile and run)
    units = n * group // tile + len(nq)
    nb = lib.d8_attention_cache_scratch_bytes(dt, len(nq), n, width, H, G, D)
    runs = (nb - 32 * units) // (4 * G * tile * ((D + 3) // 4 * 4 + 2)) - units
    tiles = [-(-m * group // tile) for m in nq]
    total = sum(t * p for t, p in zip(tiles, np_))
    mean = -(-total // sum(tiles))
    length = max(-(-total // runs), min(mean // 4 if many else mean, 4))
    assert min(length, max(np_)) >= least, (runs, length)

    r, P = np.random.default_rng(sum(np_) + D), 7
    k, v = (r.integers(-127, 128, (P, G, PAGE, D)) for _ in range(2))
    scales = 0.041 * 1.4 ** np.arange(1 - P, 1)[:, None] * np.ones(G), np.exp2(r.integers(-7, -5, (P, G)))  # (scores spread by 0.4 to 3: no page is without weight)
    cache, (kv, vv) = _pages((k, v), scales)
    # the pages of larger and larger keys, each many times, last or first or in no order; the last token of a sequence is anywhere in its page
    table, held = np.full((len(nq), width), -1, np.int32), []
    for s, p in enumerate(np_):
        at = np.sort(r.integers(0, P, p))
        table[s, :p] = at if rising == "late" else at[::-1] if rising == "early" else r.permutation(at)
        held.append(PAGE * (p - 1) + int(r.integers(1, PAGE + 1)))
    starts = np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)
    q = r.standard_normal((n, H, D)).astype(dtype)
    got, got_lse = cache.attention(q, starts, held, table, D ** -0.5, causal)
    again, again_lse = cache.attention(q, starts, held, table, D ** -0.5, causal)
    assert np.array_equal(got, again) and np.array_equal(got_lse, again_lse)
    heads = np.unique(np.r_[0, G - 1, r.integers(0, G, 2)])  # some key heads, with all that share them
    mine = (heads[:, None] * group + np.arange(group)).ravel()
    want, lse = so.attention_cache(q[:, mine], kv[:, heads], vv[:, heads], starts, held, table, P, D ** -0.5, causal)
    got, tol = f(got)[:, mine].astype(np.float64), FP16_TOL if dtype == np.float16 else FP32_TOL
    assert rel_fro(got, want) <= tol
    e, size = np.linalg.norm(got - want, axis=2), np.linalg.norm(want, axis=2)
    assert (e / (size + size.mean())).max() <= 4 * tol
    assert (np.abs(got_lse[mine] - lse) / np.maximum(1, np.abs(lse))).max() <= 1e-5
