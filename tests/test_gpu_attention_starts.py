"""d8_attention and d8_attention_grad with starts that do not rise: a start before an earlier one counts as that one, one outside the tensor as
the tensor's end, so the result is that of the starts so bounded.  Calls large enough to be cut into pieces that a second launch joins, whose
scratch is sized by the numbers of tokens: sequences that overlapped would need more of it than there is.  Tolerances as in
test_gpu_attention.py."""
import numpy as np
import pytest

import layer_oracle as lo
from test_gpu_attention import TOL, _inputs, _near

pytestmark = pytest.mark.gpu

CASES = [
    # starts of queries, of keys, queries, keys, heads, kv heads, dim
    ([0, 900, 0, 900, 300, 1200], [0, 900, 0, 900, 300, 1200], 1200, 1200, 8, 2, 64),
    ([0, 900, 0, 900], [0, 900, 0, 900], 900, 900, 8, 2, 128),                  # as many tokens as one of the two
    ([0, 1, 0, 1, 2, 0, 3], [0, 5000, 0, 5000, 9000, 0, 9100], 3, 9100, 8, 2, 64),  # single queries
    ([0, 20, 700, 10, 700], [0, 600, 100, 1 << 30, -4], 700, 800, 4, 1, 80),     # queries and keys that turn back in different places
    ([-7] + [40, 3] * 70 + [600], [-7] + [40, 3] * 70 + [600], 600, 600, 4, 2, 64),  # ... and more of them than lanes
    ([0, 300, 0, 300], [0, 300, 0, 300], 300, 300, 2, 2, 33),                   # rows that start anywhere
]


def _bounded(starts, tokens):
    return np.maximum.accumulate(np.clip(np.asarray(starts, np.int64), 0, tokens))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("cfg", range(len(CASES)))
def test_starts_that_turn_back(cfg, dtype, causal):
    from deep8_amd import ops
    qs, ks, nq, nk, H, G, D = CASES[cfg]
    q, k, v, do = _inputs([nq], [nk], H, G, D, dtype, 40 + cfg)
    wild_q, wild_k = np.asarray(qs, np.int32), np.asarray(ks, np.int32)
    qs, ks, scale = _bounded(qs, nq), _bounded(ks, nk), D ** -0.5
    want, lse = lo.attention(q, k, v, qs, ks, scale, causal)
    got, got_lse = ops.attention(q, k, v, wild_q, wild_k, scale, causal, o=np.full_like(q, 7))
    inside = ~np.isnan(want[:, 0, 0])
    _near(got[inside], want[inside], TOL[dtype])
    assert (got[~inside] == 7).all()
    seen = np.isfinite(lse)
    assert np.abs(got_lse - lse)[seen].max() <= 1e-5 * max(1, np.abs(lse[seen]).max())
    held = np.nan_to_num(got_lse, neginf=-np.inf), np.where(inside[:, None, None], got, 0).astype(dtype)
    back = ops.attention_grad(q, k, v, held[1], held[0], do, wild_q, wild_k, scale, causal)
    for g, w in zip(back, lo.attention(q, k, v, qs, ks, scale, causal, do)):
        inside = ~np.isnan(w[:, 0, 0])
        _near(g[inside], w[inside], TOL[dtype])
        assert np.isnan(g[~inside].astype(np.float32)).all()
    again = ops.attention_grad(q, k, v, held[1], held[0], do, wild_q, wild_k, scale, causal)
    assert all(np.array_equal(a, b, equal_nan=True) for a, b in zip(back, again))


def test_too_many_sequences():
    from deep8_amd import capi
    lib = capi.init()
    d, i = capi.DeviceArray((2, 32)), capi.DeviceArray.from_numpy(np.array([0, 2], np.int32))
    n = (1 << 30) + 5, 2, 2, 4, 4, 8
    assert lib.d8_attention(capi.FLOAT32, d.ptr, 32, d.ptr, 32, d.ptr, 32, d.ptr, 32, None, i.ptr, i.ptr, *n, 1.0, 1, None, 0, None) == 10001
    assert b"sequences" in lib.d8_last_error()
