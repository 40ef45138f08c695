"""d8_cache_append, d8_cache_read and d8_attention_cache against their definitions in 64 bits.

Codes, scales and values read back have one right value: equal.  Attention as d8_attention's tests: 2e-3 in Float16 (roundings to half of 2^-11 at most in
probabilities and result) and 1e-5 in Float32 (sums of up to some thousand terms, scores of up to 20 whose rounding the exponential makes a
relative error of 20 * 2^-24), relative Frobenius and per row."""
import ctypes

import numpy as np
import pytest

import serving_oracle as so
from util import FP16_TOL, FP32_TOL, f, rel_fro, rng

TOL = {np.float16: FP16_TOL, np.float32: FP32_TOL}
PAGE = 64


def _starts(n):
    return np.concatenate([[0], np.cumsum(n)]).astype(np.int32)


def _table(lengths, r, spare=3, room=0):
    """pages in no order for each sequence, -1 behind them; how many pages there are"""
    need = [-(-n // PAGE) for n in lengths]
    order, width = r.permutation(sum(need) + spare), max(need, default=0) + room
    at = np.concatenate([[0], np.cumsum(need)])
    return np.array([np.r_[order[a:a + n], [-1] * (width - n)] for a, n in zip(at, need)], np.int32).reshape(len(lengths), width), sum(need) + spare


def _rows(n, heads, dim, dtype, r, spread=True):
    x = r.standard_normal((n, heads, dim))
    if spread:  # tokens of different sizes, so that scales grow while pages fill
        x = x * np.exp2(r.integers(-3, 4, (n, 1, 1)))
    return x.astype(dtype)


def _same(cache, want, table, lengths):
    """codes and scales of every place that is held"""
    k, v, ks, vs = (a.numpy() for a in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales))
    for s, n in enumerate(lengths):
        for p in range(-(-n // PAGE)):
            page, held = table[s][p], min(n - p * PAGE, PAGE)
            assert np.array_equal(ks[page], want.scales["k"][page].astype(np.float32), equal_nan=True)
            assert np.array_equal(vs[page], want.scales["v"][page].astype(np.float32), equal_nan=True)
            assert np.array_equal(k[page, :, :held, :cache.dim], want.codes["k"][page, :, :held].astype(np.int8))
            assert np.array_equal(v[page, :, :cache.dim, :held].swapaxes(1, 2), want.codes["v"][page, :, :held].astype(np.int8))


# tokens of each sequence that come in each call; heads, dim, pad
FILLS = [([[5]], 1, 8, 0), ([[1, 1]] * 5, 2, 64, 0), ([[64, 0, 130], [1, 1, 1], [3, 70, 62]], 2, 80, 8), ([[200, 63], [1, 1], [1, 1]], 3, 128, 0), ([[17, 0, 1], [47, 64, 0], [1, 65, 129]], 1, 33, 1),
         ([[2] * 70, [1] * 70], 2, 16, 0), ([[100, 3]], 2, 256, 0), ([[90, 31], [5, 40]], 1, 7, 3), ([[300, 700]], 4, 96, 0),
         ([[70, 3], [1, 62]], 2, 100, 0), ([[70, 3], [30, 1]], 2, 64, 3), ([[5, 90], [64, 1]], 3, 44, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("calls,heads,dim,pad", FILLS)
def test_append_and_read(calls, heads, dim, pad, dtype):
    from deep8_amd import ops
    r = rng(dim + len(calls))
    lengths = np.sum(calls, 0)
    table, pages = _table(lengths, r, room=1)
    cache, want = ops.PagedCache(pages, heads, dim, fill=85), so.Cache(pages, heads, dim)
    held = np.zeros(len(lengths), np.int64)
    for new in calls:
        held += new
        starts, n = _starts(new), sum(new)
        k, v = _rows(n, heads, dim, dtype, r), _rows(n, heads, dim, dtype, r)
        cache.append(k, v, starts, held, table, pad)
        want.append(k, v, starts, held, table)
        _same(cache, want, table, held)
    for back in (held, np.minimum(held, 3), (held + 1) // 2):
        starts, n = _starts(back), int(sum(back))
        like = [np.zeros((n, heads, dim), dtype)] * 2
        for got, w in zip(cache.read(n, starts, held, table, dtype, pad), want.read(n, starts, held, table, like)):
            assert np.array_equal(got, w.astype(dtype))


@pytest.mark.gpu
def test_pages_that_are_not_there():
    """tokens without a page are left out, and read as zeros; rows of no sequence stay as they were; sequences of fewer tokens than rows; starts that turn back"""
    from deep8_amd import ops
    r = rng(4)
    table = np.array([[2, -1, 0], [7, 1, 1000], [3, 5, 4], [-5, 6, 6]], np.int32)  # 7 and 1000: no such page
    starts, lengths = np.array([2, 150, 140, 190, 200], np.int32), np.array([148, 60, 45, 300], np.int64)
    cache, want = ops.PagedCache(7, 2, 24), so.Cache(7, 2, 24)
    k, v = _rows(205, 2, 24, np.float32, r), _rows(205, 2, 24, np.float32, r)
    cache.append(k, v, starts, lengths, table)
    clean = np.maximum.accumulate(starts)
    want.append(k, v, clean, lengths, table)
    ks = cache.k_scales.numpy()
    assert np.array_equal(ks, want.scales["k"].astype(np.float32), equal_nan=True)
    like = [np.full((205, 2, 24), 9, np.float32)] * 2
    for got, w in zip(cache.read(205, starts, lengths, table, into=like), want.read(205, clean, lengths, table, like)):
        assert np.array_equal(got, w.astype(np.float32), equal_nan=True)  # (places 5 .. of a page whose first tokens were never written: no scale yet)
        assert (got[[0, 1, 200, 204]] == 9).all()


@pytest.mark.gpu
def test_tokens_that_are_no_numbers():
    from deep8_amd import ops
    r = rng(5)
    table = np.array([[0, 1]], np.int32)
    for bad in (np.nan, np.inf, -np.inf):
        cache, want = ops.PagedCache(2, 2, 16), so.Cache(2, 2, 16)
        k, v = _rows(70, 2, 16, np.float32, r), _rows(70, 2, 16, np.float32, r)
        k[10, 1, 3] = bad
        for a in (cache, want):
            a.append(k[:60], v[:60], [0, 60], [60], table)
            a.append(k[60:], v[60:], [0, 10], [70], table)
        kk, vv = cache.read(70, [0, 70], [70], table)
        assert np.isnan(kk[:64, 1]).all() and np.isfinite(kk[:, 0]).all() and np.isfinite(kk[64:]).all() and np.isfinite(vv).all()
        o, lse = cache.attention(k[:2].repeat(1, 1), [0, 2], [70], table, 0.25)
        assert np.isnan(o[:, 1]).all() and np.isfinite(o[:, 0]).all()
        # the page begins anew
        cache.append(v[:5], v[:5], [0, 5], [5], table)
        assert np.isfinite(cache.read(5, [0, 5], [5], table)[0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_largest_and_smallest_values(dtype):
    """scales at powers of two of which 127 just reach, and just do not reach, the largest element; the type's ends"""
    from deep8_amd import ops
    info = np.finfo(dtype)
    tops = [dtype(127), np.nextafter(dtype(127), dtype(200)), np.nextafter(dtype(127), dtype(0)), dtype(63.5), info.max, info.tiny, info.smallest_subnormal, dtype(0), dtype(0.7)]
    cache, want, table = ops.PagedCache(len(tops), 1, 16), so.Cache(len(tops), 1, 16), np.arange(len(tops), dtype=np.int32)[:, None]
    k = np.stack([np.concatenate([[t, -t, t / dtype(2), t / dtype(3)], np.zeros(12)]) for t in tops]).astype(dtype)[:, None]
    starts, lengths = np.arange(len(tops) + 1), np.ones(len(tops))
    cache.append(k, -k, starts, lengths, table)
    want.append(k, -k, starts, lengths, table)
    _same(cache, want, table, lengths.astype(int))
    with np.errstate(over="ignore"):
        for got, w in zip(cache.read(len(tops), starts, lengths, table, dtype), want.read(len(tops), starts, lengths, table, [k, k])):
            assert np.array_equal(got, np.clip(w, -float(info.max), float(info.max)).astype(dtype))


def _filled(lengths, heads, dim, r, spare=2, size=1.0):
    """a cache of random codes, and its values [page][head][token][dim]"""
    from deep8_amd import ops
    table, pages = _table(lengths, r, spare)
    cache = ops.PagedCache(pages, heads, dim)
    out = []
    for name in "kv":
        codes = r.integers(-128, 128, (pages, heads, PAGE, cache.pitch), dtype=np.int8)
        scales = (np.exp2(r.integers(-8, -4, (pages, heads))) * size * np.where(r.random((pages, heads)) < 0.5, 1, 1.37)).astype(np.float32)
        getattr(cache, name + "_codes").copy_from(codes if name == "k" else np.ascontiguousarray(codes.swapaxes(2, 3)))
        getattr(cache, name + "_scales").copy_from(scales)
        out.append(codes[..., :dim].astype(np.float64) * scales[..., None, None])
    return cache, table, pages, out


def _near(got, want, tol):
    got, want = f(got).astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    if not want.size:
        return
    assert rel_fro(got, want) <= tol
    e, n = np.linalg.norm((got - want).reshape(len(want), -1), axis=1), np.linalg.norm(want.reshape(len(want), -1), axis=1)
    assert (e <= 4 * tol * (n + n.mean())).all()


ATTENTION = [
    # queries and tokens of each sequence, heads, kv heads, dim, causal, pad
    ([1], [1], 1, 1, 8, True, 0),
    ([1, 1, 1], [300, 1, 64], 8, 2, 128, True, 0),              # decoding
    ([1, 1], [900, 1000], 5, 1, 96, True, 8),
    ([1], [9000], 4, 4, 64, True, 0),                           # one long sequence: many runs to join
    ([1] * 70, [3] * 69 + [700], 2, 2, 32, True, 0),            # more sequences than lanes of a wave
    ([5, 0, 3], [70, 50, 2], 4, 2, 80, True, 0),                # queries that see nothing, a sequence without any
    ([4, 2], [0, 0], 2, 1, 32, True, 0),                        # no keys at all
    ([33, 20], [33, 500], 6, 2, 64, True, 0),                   # several tiles of few rows
    ([130, 64, 1], [130, 700, 300], 8, 2, 128, True, 0),        # many rows a sequence
    ([128, 256], [128, 300], 4, 4, 64, True, 0),
    ([100], [1500], 16, 1, 128, True, 16),
    ([70, 90], [50, 200], 4, 1, 64, False, 0),                  # another sequence's states
    ([300, 5], [77, 129], 3, 3, 112, False, 0),
    ([50], [50], 3, 1, 33, True, 3),                            # rows that start anywhere
    ([3, 200], [64, 230], 2, 2, 7, True, 1),
    ([20, 70], [20, 170], 2, 1, 256, True, 0),                  # the widest heads
    ([20, 70], [20, 170], 2, 1, 200, False, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("nq,nk,H,G,D,causal,pad", ATTENTION)
def test_attention(nq, nk, H, G, D, causal, pad, dtype):
    r = rng(sum(nq) + D)
    cache, table, pages, (kv, vv) = _filled(nk, G, D, r)
    q, starts = r.standard_normal((sum(nq), H, D)).astype(dtype), _starts(nq)
    want, lse = so.attention_cache(q, kv, vv, starts, nk, table, pages, D ** -0.5, causal)
    got, got_lse = cache.attention(q, starts, nk, table, D ** -0.5, causal, pad)
    _near(got, want, TOL[dtype])
    empty = np.isneginf(lse)
    assert np.array_equal(np.isneginf(got_lse), empty) and (f(got)[empty.T] == 0).all()
    assert np.abs(got_lse[~empty] - lse[~empty]).max(initial=0) <= 1e-5 * max(1, np.abs(lse[~empty]).max(initial=0))
    again, again_lse = cache.attention(q, starts, nk, table, D ** -0.5, causal, pad)
    assert np.array_equal(got, again) and np.array_equal(got_lse, again_lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_attention_with_pages_and_rows_left_out(dtype):
    """rows before, between and behind sequences; tables with holes, ids out of range, too short for the lengths"""
    r = rng(8)
    cache, _, pages, (kv, vv) = _filled([400], 2, 48, r)
    table = np.array([[3, -1, 0, 900], [1, 2, 4, 5], [-7, -1, 99, 7], [6, 6, 6, 6]], np.int32)
    starts, lengths = np.array([2, 7, 90, 93, 95], np.int32), np.array([250, 900, 130, 64], np.int64)
    q = r.standard_normal((100, 4, 48)).astype(dtype)
    before = np.full_like(q, 3)
    for causal in (True, False):
        want, lse = so.attention_cache(q, kv, vv, starts, lengths, table, pages, 0.2, causal)
        got, got_lse = cache.attention(q, starts, lengths, table, 0.2, causal, o=before)
        mine = slice(2, 95)
        assert (got[:2] == 3).all() and (got[95:] == 3).all() and np.isnan(got_lse[:, :2]).all() and np.isnan(got_lse[:, 95:]).all()
        _near(got[mine], want[mine], TOL[dtype])
        empty = np.isneginf(lse[:, mine])
        assert np.array_equal(np.isneginf(got_lse[:, mine]), empty)
        back = np.array([2, 7, 5, 93, 95], np.int32)  # a start that turns back counts as the one before it
        a, b = cache.attention(q, back, lengths, table, 0.2, causal, o=before), cache.attention(q, np.maximum.accumulate(back), lengths, table, 0.2, causal, o=before)
        assert all(np.array_equal(x, y, equal_nan=True) for x, y in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("nq", [[1, 1], [80, 150]])
def test_pages_out_of_scale_beside_others(nq, dtype):
    """values of one page 2^20 times the others', where a sequence's queries give it next to no weight: what the others hold keeps its bits"""
    r = rng(9)
    nk = [400, 300]
    cache, table, pages, (kv, vv) = _filled(nk, 2, 64, r)
    q = np.abs(r.standard_normal((sum(nq), 4, 64))).astype(dtype)
    for s in range(2):  # the first page: keys far against the queries, values large
        p = table[s][0]
        k, ks, vs = cache.k_codes.numpy(), cache.k_scales.numpy(), cache.v_scales.numpy()
        k[p] = -100
        ks[p], vs[p] = 0.5, vs[p] * 2.0 ** 20
        cache.k_codes.copy_from(k), cache.k_scales.copy_from(ks), cache.v_scales.copy_from(vs)
        kv[p], vv[p] = -50.0, vv[p] * 2.0 ** 20
    starts = _starts(nq)
    want, _ = so.attention_cache(q, kv, vv, starts, nk, table, pages, 0.125, False)
    got, _ = cache.attention(q, starts, nk, table, 0.125, False)
    assert np.abs(want).max() < 100
    _near(got, want, TOL[dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("n", [16, 130])
def test_scores_small_and_large_side_by_side(n, dtype):
    """rows whose largest scores are 1, some hundred, some thousand and 2^24 and more, in turn.  A score, a sum of 64 products, is off by 64 E of the products'
    absolute sum at most, E = 2^-24, and a weight by the exponential of twice that: rows where that says nothing are the ones with one key far above all
    others, whose weights are 1 and 0 in any case"""
    r = rng(31)
    cache, table, pages, (kv, vv) = _filled([300], 1, 64, r)
    size = np.array([1, 300, 900, 1100, 5000])[np.arange(n) % 5]
    q = r.standard_normal((n, 1, 64)) * (size / 20)[:, None, None]
    q = q.astype(np.float16).astype(dtype)
    scale = 0.125
    if dtype == np.float32:
        q[7] *= 2.0 ** 16
    want, lse = so.attention_cache(q, kv, vv, [0, n], [300], table, pages, scale, False)
    got, got_lse = cache.attention(q, [0, n], [300], table, scale, False)
    got = f(got)[:, 0].astype(np.float64)
    keys = np.concatenate([kv[p, 0] for p in table[0]])[:300]
    values = np.concatenate([vv[p, 0] for p in table[0]])[:300]
    terms = scale * (np.abs(f(q)[:, 0].astype(np.float64)) @ np.abs(keys).T)
    off = np.expm1(np.minimum(2 * 64 * 2.0 ** -24 * terms.max(1), 1.0))
    score = np.sort(scale * (f(q)[:, 0].astype(np.float64) @ keys.T), 1)
    alone = score[:, -1] - score[:, -2] > 40 + 4 * 64 * 2.0 ** -24 * terms.max(1)
    bound = np.where(alone, 0, 2 * off * np.abs(values).max()) + 4 * TOL[dtype] * np.abs(values).max()
    assert np.isfinite(got).all() and np.isfinite(got_lse).all()
    assert (np.abs(got - want[:, 0]).max(1) <= bound).all()
    assert (np.abs(got_lse - lse) <= 64 * 2.0 ** -24 * terms.max(1) + 1e-5 * np.maximum(1, np.abs(lse))).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [6, 96])
def test_queries_of_any_size(n):
    """rows of 1e-37 to 1e37, elements of different sizes in a row, rows of zeros; one with an infinity and one with NaN, which stay theirs alone"""
    r = rng(12)
    cache, table, pages, (kv, vv) = _filled([200], 1, 64, r)
    q = r.standard_normal((n, 1, 64))
    size = np.array([1e-37, 1e-20, 1.0, 1e20, 1e37, 0.0])
    q = (q * size[np.arange(n) % 6][:, None, None]).astype(np.float32)
    q[2] *= np.exp2(-r.integers(0, 40, 64))
    want, lse = so.attention_cache(q, kv, vv, [0, n], [200], table, pages, 0.125, False)
    got, got_lse = cache.attention(q, [0, n], [200], table, 0.125, False)
    _near(got, want, FP32_TOL)
    assert (np.abs(got_lse - lse) <= 1e-5 * np.maximum(1, np.abs(lse))).all()
    q[3, 0, 5], q[5, 0, 9] = np.inf, np.nan
    bad, _ = cache.attention(q, [0, n], [200], table, 0.125, False)
    rest = np.ones(n, bool)
    rest[[3, 5]] = False
    assert np.array_equal(bad[rest], got[rest]) and np.isnan(bad[[3, 5]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [[1, 1, 1], [40, 3, 90]])
def test_steps_captured_and_replayed(nq):
    """an append and the attention after it, captured once; lengths, tokens and queries change between the replays, eager calls run between them"""
    from deep8_amd import capi, ops
    lib, r, H, G, D, dtype = capi.init(), rng(10), 8, 2, 64, np.float16
    longest = [500, 90, 300]
    table, pages = _table(longest, r)
    starts, n = _starts(nq), sum(nq)
    live, other = ops.PagedCache(pages, G, D), ops.PagedCache(pages, G, D)
    held = np.array([300, 0, 128])
    first = [_rows(int(held.sum()), G, D, dtype, r, False) for _ in range(2)]
    for c in (live, other):
        c.append(*first, _starts(held), held, table)
    d = {name: capi.DeviceArray((n, h, D), dtype) for name, h in (("q", H), ("k", G), ("v", G), ("o", H))}
    lse, ints = capi.DeviceArray((H, n)), {"starts": capi.DeviceArray.from_numpy(starts), "lengths": capi.DeviceArray((3,), np.int32), "table": capi.DeviceArray.from_numpy(table)}
    where = (*(ints[i].ptr for i in ("starts", "lengths", "table")), 3, n, table.shape[1], pages)
    nb = lib.d8_attention_cache_scratch_bytes(capi.FLOAT16, 3, n, table.shape[1], H, G, D)
    ws = capi.DeviceArray((nb,), np.uint8)
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    capi.check(lib.d8_stream_create(ctypes.byref(stream)))
    capi.check(lib.d8_graph_begin(stream))
    rcs = [lib.d8_cache_append(capi.FLOAT16, d["k"].ptr, G * D, d["v"].ptr, G * D, *live._state(), *where, G, D, stream),
           lib.d8_attention_cache(capi.FLOAT16, d["q"].ptr, H * D, *live._state(), d["o"].ptr, H * D, lse.ptr, *where, H, G, D, 0.125, 1, ws.ptr, nb, stream)]
    capi.check(lib.d8_graph_end(stream, ctypes.byref(graph)))
    assert rcs == [0, 0]
    for _ in range(2):
        held = held + nq
        q, k, v = (_rows(n, h, D, dtype, r, False) for h in (H, G, G))
        for name, x in (("q", q), ("k", k), ("v", v)):
            d[name].copy_from(x)
        ints["lengths"].copy_from(held.astype(np.int32))
        capi.check(lib.d8_graph_launch(graph, stream))
        capi.sync(stream)
        other.append(k, v, starts, held, table)
        want, want_lse = other.attention(q, starts, held, table, 0.125)
        assert np.array_equal(d["o"].numpy(), want) and np.array_equal(lse.numpy(), want_lse)
    capi.check(lib.d8_graph_destroy(graph))
    capi.check(lib.d8_stream_destroy(stream))


@pytest.mark.gpu
def test_a_cache_that_passes_4_gib():
    """offsets of codes beyond 32 bits: tokens written and read at the last of many pages"""
    from deep8_amd import capi, ops
    r, G, D = rng(11), 16, 256
    pages = (1 << 32) // (G * D * PAGE) + 70
    free, total = ctypes.c_size_t(), ctypes.c_size_t()
    capi.check(capi.init().d8_mem_info(ctypes.byref(free), ctypes.byref(total)))
    if free.value < 12 << 30:
        pytest.skip("not enough device memory")
    cache = ops.PagedCache.__new__(ops.PagedCache)
    cache.pages, cache.kv_heads, cache.dim, cache.pitch = pages, G, D, D
    cache.k_codes, cache.v_codes = (capi.DeviceArray((pages, G, PAGE, D), np.int8) for _ in range(2))
    cache.k_scales, cache.v_scales = (capi.DeviceArray.from_numpy(np.full((pages, G), np.nan, np.float32)) for _ in range(2))
    table, n = np.array([[0, pages - 1, 1, pages - 2]], np.int32), 4 * PAGE - 9
    k, v = (r.standard_normal((n, G, D)).astype(np.float16) for _ in range(2))
    cache.append(k, v, [0, n], [n], table)
    small, small_table = ops.PagedCache(4, G, D), np.array([[0, 1, 2, 3]], np.int32)
    small.append(k, v, [0, n], [n], small_table)
    for a, b in zip(cache.read(n, [0, n], [n], table), small.read(n, [0, n], [n], small_table)):
        assert np.array_equal(a, b)
    for m in (1, 100):
        q = r.standard_normal((m, 2 * G, D)).astype(np.float16)
        for a, b in zip(cache.attention(q, [0, m], [n], table, 0.0625), small.attention(q, [0, m], [n], small_table, 0.0625)):
            assert np.array_equal(a, b)


@pytest.mark.gpu
def test_nothing_to_do():
    from deep8_amd import ops
    cache = ops.PagedCache(2, 1, 16)
    none, q = np.zeros((0, 1, 16), np.float32), np.ones((3, 1, 16), np.float32)
    cache.append(none, none, [0, 0], [0], [[0]])
    assert cache.read(0, [0, 0], [0], [[0]])[0].shape == (0, 1, 16)
    assert cache.attention(none, [0, 0], [5], [[0]], 1.0)[0].shape == (0, 1, 16)
    # a table without room: nothing to see, and nothing read
    o, lse = cache.attention(q, [0, 3], [5], np.zeros((1, 0)), 1.0)
    assert not o.any() and np.isneginf(lse).all()
    cache.append(q, q, [0, 3], [5], np.zeros((1, 0)))
    assert not cache.read(3, [0, 3], [5], np.zeros((1, 0)), into=(q, q))[0].any()
    # no sequences: every row left alone
    assert (cache.attention(q, [0], [], np.zeros((0, 1)), 1.0, o=q)[0] == 1).all()


def test_refusals():
    """(refused before anything is launched: the tensors need not be there, nor a device)"""
    from deep8_amd import capi
    lib, p, big = capi.load(), 64, 1 << 40

    def refused(fn, good, cases, code=10001):
        for i, v in cases:
            a = list(good)
            a[i] = v
            assert fn(*a) == code, (fn.__name__, i, v)
    rows = (capi.FLOAT16, p, 64, p, 64, p, p, p, p, p, p, p, 2, 3, 4, 5, 2, 32, None)
    for fn in (lib.d8_cache_append, lib.d8_cache_read):
        refused(fn, rows, [(1, None), (2, 63), (3, None), (4, 63), (5, None), (5, 72), (6, None), (7, None), (7, 8), (8, None), (9, None), (10, None), (11, None), (12, -1), (13, -1), (14, -1),
                           (15, -1), (16, 0), (17, 0), (17, 257), (12, 1 << 24), (14, 1 << 24), (13, 1 << 30)])
        refused(fn, rows, [(0, capi.FLOAT64), (0, 3)], 10002)
        assert fn(*rows[:12], 1 << 23, 1 << 23, *rows[14:]) == 10001  # 2^24 pages and heads, of 256 threads each
    att = (capi.FLOAT16, p, 128, p, p, p, p, p, 128, p, p, p, p, 2, 3, 4, 5, 4, 2, 32, 0.5, 1, p, big, None)
    refused(lib.d8_attention_cache, att, [(1, None), (2, 127), (3, None), (3, 72), (4, None), (5, None), (6, None), (7, None), (8, 127), (10, None), (11, None), (12, None), (13, -1), (14, -1), (15, -1),
                                          (16, -1), (17, 3), (17, 1), (18, 0), (19, 0), (19, 257), (20, float("nan")), (22, None), (22, 72), (23, 0)])
    refused(lib.d8_attention_cache, att, [(0, capi.FLOAT64)], 10002)
    assert lib.d8_attention_cache(*att[:13], 1 << 23, 1 << 23, *att[15:]) == 10001
    size = lib.d8_attention_cache_scratch_bytes
    assert size(capi.FLOAT16, 2, 3, 4, 4, 2, 32) > 0
    assert [size(*a) for a in ((capi.FLOAT64, 2, 3, 4, 4, 2, 32), (capi.FLOAT16, 2, 3, 4, 3, 2, 32), (capi.FLOAT16, 2, 3, -1, 4, 2, 32), (capi.FLOAT16, 2, 3, 4, 4, 2, 300))] == [0] * 4


@pytest.mark.parametrize("sequences,tokens,table_pages,heads,kv_heads,dim", [(1, 1, 100000, 8, 8, 128), (500, 500, 64, 32, 8, 128), (3, 5000, 200, 16, 2, 64), (2, 2, 1, 1, 1, 16)])
def test_scratch_has_room_for_every_piece(sequences, tokens, table_pages, heads, kv_heads, dim):
    """a model of how the device cuts the work, over random lengths: slots (run + tile) are never shared, and lie in what was asked for"""
    from deep8_amd import capi
    lib, group, r = capi.load(), heads // kv_heads, rng(tokens)
    for dt in (capi.FLOAT16, capi.FLOAT32):
        nb = lib.d8_attention_cache_scratch_bytes(dt, sequences, tokens, table_pages, heads, kv_heads, dim)
        many = dim <= 128 and tokens * group // min(sequences, tokens) >= (33 if dt == capi.FLOAT16 else 96)
        rows = 128 if many else 16
        units = tokens * group // rows + min(sequences, tokens)
        per_slot = 4 * kv_heads * rows * ((dim + 3) // 4 * 4 + 2)
        slots = (nb - 32 * units) // per_slot  # (32 bytes a tile say what is joined)
        runs = slots - units
        assert runs >= 1 and nb == 32 * units + slots * per_slot
        for _ in range(20):
            cuts = np.sort(r.integers(0, tokens + 1, sequences - 1))
            n = np.diff(np.r_[0, cuts, tokens])
            pages = np.maximum(1, r.integers(0, table_pages + 1, sequences))
            tiles = -(-n * group // rows)
            assert tiles.sum() <= units
            total = int((tiles * pages).sum())
            mean = -(-total // int(tiles.sum()))
            length = max(-(-total // runs), min(mean // 4 if many else mean, 4))
            used, at, unit = set(), 0, 0
            for t, p in zip(tiles, pages):
                for _ in range(t):
                    for run in range(at // length, (at + int(p) - 1) // length + 1):
                        assert run < runs and run + unit < slots and (run + unit) not in used
                        used.add(run + unit)
                    at, unit = at + int(p), unit + 1
