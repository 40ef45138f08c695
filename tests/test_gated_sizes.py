"""How long the rows of d8_matmul_gated may be: tiles are addressed by 32 bits, so 128 rows of x (fewer if there are fewer) and a step's rows of w
must fit in 2 GiB; what does not is refused, by the scratch query too, and what just fits is right."""
import numpy as np
import pytest

import layer_oracle as lo
from util import FP16_TOL, FP32_TOL, f, rel_fro, rng

# rows, inner, cols of the first size that is refused
X_LIMITS = {"float32": [(128, (1 << 22) + 1, 4), (5000, (1 << 22) + 1, 8), (65, 8259553, 4), (2, (1 << 28) + 1, 4)],
            "float16": [(128, (1 << 23) + 1, 8), (65, 16519105, 8)]}
W_LIMITS = {"float32": [(1, 64, (1 << 23) + 1), (500, 64, (1 << 23) + 1)], "float16": [(64, 64, (1 << 24) + 1), (65, 8, (1 << 23) + 1)]}


def _cases():
    for name in ("float32", "float16"):
        for i, limits in enumerate((X_LIMITS, W_LIMITS)):
            for size in limits[name]:
                yield name, i, size


@pytest.mark.parametrize("name,which,size", _cases())
def test_scratch_query(name, which, size):
    from deep8_amd import capi
    lib, dt = capi.load(), {"float32": capi.FLOAT32, "float16": capi.FLOAT16}[name]
    rows, inner, cols = size
    assert lib.d8_matmul_gated_scratch_bytes(dt, 0, rows, inner, cols) == 0
    # an ordinary number of rows of an ordinary length asks for what it did: parts of the sums of few rows
    assert lib.d8_matmul_gated_scratch_bytes(dt, 0, 4, 4096, 512) > 0


@pytest.mark.gpu
@pytest.mark.parametrize("name,which,size", _cases())
def test_refused(name, which, size):
    from deep8_amd import capi
    lib, dt = capi.init(), {"float32": capi.FLOAT32, "float16": capi.FLOAT16}[name]
    rows, inner, cols = size
    d = capi.DeviceArray((64,))
    # (refused before anything is launched: the tensors need not be there)
    assert lib.d8_matmul_gated(dt, d.ptr, rows, inner, d.ptr, cols, 0, None, d.ptr, d.ptr, 1 << 60, None) == 10001
    if inner < 1 << 28 and cols < 1 << 28:
        assert b"too long" in lib.d8_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,inner,cols", [(np.float32, 128, 1 << 22, 4), (np.float16, 70, 15339168, 8), (np.float32, 3, 40, 1 << 23), (np.float16, 66, 72, 1 << 23)])
def test_longest_rows(dtype, rows, inner, cols):
    """a thousand elements of x and w among zeros, the last of each row and column with them"""
    from deep8_amd import ops
    r = rng(rows)
    k = np.unique(np.r_[r.integers(0, inner, 1000), 0, inner - 1])
    n = np.unique(np.r_[r.integers(0, cols, 1000), 0, cols - 1])
    x, w = np.zeros((rows, inner), dtype), np.zeros((inner, 2 * cols), dtype)
    x[:, k] = r.standard_normal((rows, len(k)))
    both = np.r_[n, n + cols]
    w[np.ix_(k, both)] = r.standard_normal((len(k), len(both))) * len(k) ** -0.5
    want, _ = lo.gated(x[:, k], w[np.ix_(k, both)], "silu")
    got, _ = ops.matmul_gated(x, w, keep=False)
    rest = np.ones(cols, bool)
    rest[n] = False
    assert rel_fro(f(got[:, n]), want) <= (FP16_TOL if dtype == np.float16 else FP32_TOL)
    assert not got[:, rest].any()
