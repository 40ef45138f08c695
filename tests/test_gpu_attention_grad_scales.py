"""d8_attention_grad beside rows of another size: the score's gradient is held in half relative to a bound, and rows that a sum has nothing to do
with must not move it.  NaN, infinities and the largest halves in other sequences, in rows of no sequence and in other key heads must leave
a sequence's gradients as they are without them, and a row's dq does not lose bits to the rows beside it.  Tolerances as in
test_gpu_attention.py: the same roundings."""
import numpy as np
import pytest

import layer_oracle as lo
from test_gpu_attention import TOL, _inputs, _near, _starts
from util import f

pytestmark = pytest.mark.gpu

SIZES = [
    # lengths, heads, kv heads, dim, pad
    ([20, 45, 9, 300], 4, 2, 64, 0),
    ([20, 45, 9, 300], 4, 2, 128, 8),
    ([20, 45, 9, 60], 2, 2, 33, 1),          # rows that start anywhere
    ([700, 300, 9, 1200], 8, 2, 128, 0),     # rows in chunks that a second launch joins
    ([20, 45, 9, 300], 2, 1, 200, 0),
]


@pytest.mark.parametrize("bad", [np.inf, np.nan, 6e4, -6e4])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_rows_of_other_sequences(size, dtype, bad):
    from deep8_amd import ops
    lengths, H, G, D, pad = SIZES[size]
    q, k, v, do = _inputs(lengths, lengths, H, G, D, dtype, 50 + size)
    s, scale = _starts(lengths), D ** -0.5
    # the second sequence and the last rows, which are of no sequence, hold what is out of scale
    wild = v.copy(), do.copy()
    for a in wild:
        a[s[1]:s[2]], a[s[3] + lengths[3] // 2:] = bad, bad
    starts = s.copy()
    starts[4] = s[3] + lengths[3] // 2
    for causal in (True, False):
        want = lo.attention(q, k, v, starts, starts, scale, causal, do)
        o, lse = ops.attention(q, k, v, starts, starts, scale, causal)
        o[s[1]:s[2]], o[starts[4]:] = 1, 1
        got = ops.attention_grad(q, k, wild[0], o, np.nan_to_num(lse), wild[1], starts, starts, scale, causal, pad=pad)
        for g, w in zip(got, want):
            for part in (slice(0, s[1]), slice(s[2], s[3]), slice(s[3], starts[4])):
                _near(g[part], w[part], TOL[dtype])


@pytest.mark.parametrize("which", ["v", "do"])
@pytest.mark.parametrize("size", range(len(SIZES)))
def test_another_key_head(size, which):
    """the heads that share other keys have values or output gradients of 6 10^4"""
    from deep8_amd import ops
    lengths, H, G, D, pad = SIZES[size]
    if G == 1:
        H, G = 2, 2
    q, k, v, do = _inputs(lengths, lengths, H, G, D, np.float16, 60 + size)
    s, scale = _starts(lengths), D ** -0.5
    (v if which == "v" else do)[:, (G if which == "v" else H) // 2:] = 6e4
    want = lo.attention(q, k, v, s, s, scale, True, do)
    o, lse = lo.attention(q, k, v, s, s, scale, True)
    got = ops.attention_grad(q, k, v, o.astype(np.float16), lse.astype(np.float32), do, s, s, scale, True, pad=pad)
    for g, w, n in zip(got, want, (H, G, G)):
        _near(g[:, : n // 2], w[:, : n // 2], TOL[np.float16])


@pytest.mark.parametrize("D,pad", [(64, 0), (128, 0), (33, 1)])
def test_a_large_row_beside_small_ones(D, pad):
    """output gradients of 1 beside one of 6 10^4 in the same sequence, over 4096 keys: each row's dq keeps its bits"""
    from deep8_amd import ops
    q, k, v, do = _inputs([96], [4096], 2, 1, D, np.float16, 70)
    do[40] = 6e4
    qs, ks, scale = _starts([96]), _starts([4096]), D ** -0.5
    o, lse = ops.attention(q, k, v, qs, ks, scale, False)
    want = lo.attention(q, k, v, qs, ks, scale, False, do)[0]
    got = ops.attention_grad(q, k, v, o, lse, do, qs, ks, scale, False, pad=pad)[0]
    rest = np.arange(96) != 40
    _near(got[rest], want[rest], TOL[np.float16])


def test_an_infinite_row_of_the_same_sequence():
    """a query whose output gradient is infinite: its own dq and the gradients of the keys that it sees are no number, the other queries' dq and
    the keys of later queries only (here beyond its tiles) are what they are without it"""
    from deep8_amd import ops
    q, k, v, do = _inputs([600], [600], 2, 1, 64, np.float16, 71)
    s, scale = _starts([600]), 0.125
    o, lse = ops.attention(q, k, v, s, s, scale, True)
    want = lo.attention(q, k, v, s, s, scale, True, do)
    do[30] = np.inf
    dq, dk, dv = ops.attention_grad(q, k, v, o, lse, do, s, s, scale, True)
    rest = np.arange(600) != 30
    _near(dq[rest], want[0][rest], TOL[np.float16])
    assert not np.isfinite(f(dq[30])).any() and not np.isfinite(f(dk[:31])).all(axis=(1, 2)).any()
    for g, w in ((dk, want[1]), (dv, want[2])):
        _near(g[256:], w[256:], TOL[np.float16])
