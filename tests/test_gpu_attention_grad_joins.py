"""d8_attention_grad where the rows that dk and dv walk are cut into chunks whose sums a second launch joins: heads of 128, which keep fragments of
the values in LDS, on workgroups of 64 keys and of 128 (from 512 blocks of 128 keys of all key heads on).  Tolerances as in
test_gpu_attention.py."""
import functools

import numpy as np
import pytest

import layer_oracle as lo
from test_gpu_attention import TOL, _inputs, _near, _starts

pytestmark = pytest.mark.gpu

CASES = [
    # queries, keys of each sequence, heads, kv heads, dim, causal
    ([900, 300], [900, 300], 8, 2, 128, True),       # 64 keys a workgroup, up to 8 chunks of 512 rows
    ([900, 300], [900, 300], 8, 2, 128, False),
    ([1100, 40], [700, 900], 6, 2, 104, True),       # rows that see no key of some blocks
    ([700, 650], [700, 650], 2, 2, 128, True),       # heads of their own: chunks of one head's rows
    ([800], [8065], 16, 8, 100, True),               # 128 keys a workgroup, two chunks
    ([800], [8065], 16, 8, 100, False),
]


@functools.lru_cache(maxsize=1)
def _case(i):
    nq, nk, H, G, D, causal = CASES[i]
    q, k, v, do = _inputs(nq, nk, H, G, D, np.float16, 80 + i)
    qs, ks, scale = _starts(nq), _starts(nk), D ** -0.5
    o, lse = lo.attention(q, k, v, qs, ks, scale, causal)
    return (q, k, v, do, o, lse), (qs, ks, scale, causal), lo.attention(q, k, v, qs, ks, scale, causal, do)


@pytest.mark.parametrize("i,dtype", [(i, t) for i in range(len(CASES)) for t in (np.float16, np.float32)])
def test_chunks_are_joined(i, dtype):
    from deep8_amd import ops
    (q, k, v, do, o, lse), args, want = _case(i)
    q, k, v, do, o = (a.astype(dtype) for a in (q, k, v, do, o))
    got = ops.attention_grad(q, k, v, o, lse.astype(np.float32), do, *args)
    for g, w in zip(got, want):
        _near(g, w, TOL[dtype])
    again = ops.attention_grad(q, k, v, o, lse.astype(np.float32), do, *args)
    assert all(np.array_equal(a, b) for a, b in zip(got, again))
    # added to ones: the sum is rounded once more, to 2^-11 (2^-24) of about 1
    summed = ops.attention_grad(q, k, v, o, lse.astype(np.float32), do, *args, into=[np.ones_like(a) for a in got])
    for s, w in zip(summed, want):
        _near(s, w + 1, TOL[dtype])
