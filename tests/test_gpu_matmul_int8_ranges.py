"""d8_matmul_int8 with scales from 2^-100 up to what a row of the largest numbers has, whose product may be outside single precision where the result is not.

z is off by three roundings, of the sum, and of its product with one scale and then the other: 3 * 2^-24, or half a step where numbers are 2^-149 apart (half: and
by its own)."""
import numpy as np
import pytest

from util import rng

# few rows (one part, several), tiles of 64 x 64 (one part, several; rows of z four elements at a time, and not), tiles of 256 x 256
SIZES = [(5, 130, 40), (3, 16384, 40), (40, 200, 33), (70, 300, 130), (70, 300, 131), (66, 8192, 64), (4096, 128, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,inner,cols", SIZES)
def test_scales_of_any_size(rows, inner, cols, dtype):
    from deep8_amd import ops
    r, pitch = rng(rows + inner), (inner + 127) // 128 * 128
    x, w = (np.pad(r.integers(-128, 128, (n, inner), dtype=np.int8), ((0, 0), (0, pitch - inner))) for n in (rows, cols))
    x[rows // 2], w[cols // 2] = 0, 0  # sums of zero, whatever the scales are

    def scales(n):
        e = np.where(r.random(n) < 0.5, r.integers(-100, 121, n), r.integers(-80, -60, n))
        s = np.ldexp(1 + r.random(n), e).astype(np.float32)
        s[::7] *= -1
        return s
    xs, ws = scales(rows), scales(cols)
    xs[:4], ws[:4] = [2.0 ** -75, 2.0 ** -100, 2.0 ** 120, 1][:rows], [2.0 ** -75, 2.0 ** 120, 2.0 ** 120, 2.0 ** -100]
    got = ops.matmul_int8(x, xs, w, ws, inner, dtype).astype(np.float64)
    sums = x.astype(np.float32) @ w.astype(np.float32).T if inner < 1000 else x.astype(np.float64) @ w.astype(np.float64).T  # (2^14 * 1000 < 2^24)
    want = sums.astype(np.float64) * (xs.astype(np.float64)[:, None] * ws.astype(np.float64))
    most = float(np.finfo(dtype).max)
    big = np.abs(want) > most * (1 - 2.0 ** -10)
    step, half = (2.0 ** -25, 2.0 ** -11) if dtype == np.float16 else (2.0 ** -150, 0)
    bound = (half + 3 * 2.0 ** -24) * np.abs(want) + step
    assert not np.isnan(got).any()
    assert (np.abs(got - want) <= bound)[~big].all()
    assert np.array_equal(np.sign(got[big]), np.sign(want[big])) and (np.abs(got[big]) >= most * (1 - 2.0 ** -9)).all()
    assert not got[rows // 2].any() and not got[:, cols // 2].any()
