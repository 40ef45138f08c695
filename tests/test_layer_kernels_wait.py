"""The wait states of test_kernel_wait_states.py in the kernels of attention and the gated product, whose loads into LDS are asm too."""
import concurrent.futures
import struct

import pytest

from deep8_amd import capi
from test_kernel_registers import _code_objects
from test_kernel_wait_states import OBJDUMP, _check

NAMES = (b"gated_wide_kernel", b"gated_tile_kernel", b"attention_rows_kernel", b"attention_grad_kv_kernel")


def _blob():
    with open(capi.LIB_PATH, "rb") as f:
        return f.read()


@pytest.mark.skipif(OBJDUMP is None, reason="llvm-objdump is not installed")
def test_loads_into_lds_wait_for_their_scalars(tmp_path):
    blob, paths = _blob(), []
    for at in _code_objects(blob):
        shoff, = struct.unpack_from("<Q", blob, at + 40)
        shentsize, shnum = struct.unpack_from("<HH", blob, at + 58)
        image = blob[at:at + shoff + shentsize * shnum]
        if any(n in image for n in NAMES):
            paths.append(tmp_path / f"{at}.elf")
            paths[-1].write_bytes(image)
    if not paths:
        pytest.skip("the library's code objects are compressed")
    with concurrent.futures.ProcessPoolExecutor(4) as pool:
        checked = list(pool.map(_check, paths))
    loads, wrong = sum(n for n, _ in checked), [w for _, some in checked for w in some]
    assert loads > 1000
    assert not wrong, f"{len(wrong)} of {loads} loads: {wrong[:3]}"

