"""The wait states of test_kernel_wait_states.py in the product in 8-bit integers, which has the tile loop of the large product and so its asm loads."""
import struct

import pytest

from deep8_amd import capi
from test_kernel_registers import _code_objects
from test_kernel_wait_states import OBJDUMP, _check


@pytest.mark.skipif(OBJDUMP is None, reason="llvm-objdump is not installed")
def test_loads_into_lds_wait_for_their_scalars(tmp_path):
    with open(capi.LIB_PATH, "rb") as f:
        blob = f.read()
    checked = []
    for at in _code_objects(blob):
        shoff, = struct.unpack_from("<Q", blob, at + 40)
        shentsize, shnum = struct.unpack_from("<HH", blob, at + 58)
        image = blob[at:at + shoff + shentsize * shnum]
        if b"int8_wide_kernel" in image:
            path = tmp_path / f"{at}.elf"
            path.write_bytes(image)
            checked.append(_check(path))
    if not checked:
        pytest.skip("the library's code objects are compressed")
    loads, wrong = sum(n for n, _ in checked), [w for _, some in checked for w in some]
    assert loads > 200
    assert not wrong, f"{len(wrong)} of {loads} loads: {wrong[:3]}"
