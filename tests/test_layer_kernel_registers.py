"""Registers of a transformer layer's kernels, read from the code objects of the built library: which hold everything in registers, and which are
known to be short of some and keep no more than that in scratch memory."""
import re

import pytest

from deep8_amd import capi
from test_kernel_registers import _code_objects, _kernels

# (kernel, half or single, padded head, SPLIT or waves): registers in scratch memory at most; others none
SHORT = {("attention_grad_kv_kernel", "half", 128, 1): 3, ("attention_grad_kv_kernel", "half", 64, 1): 3}
WIDEST = 256  # heads above 128: not tuned


def _found():
    with open(capi.LIB_PATH, "rb") as f:
        blob = f.read()
    for at in _code_objects(blob):
        for k in _kernels(blob, at):
            m = re.search(r"\d((?:attention|gated|head_norm)_\w*?kernel)(?:I(DF16_|f)(?:Li(\d+)E)?(?:Li(\d+)E)?)?", k[".name"])
            if m:
                yield (m[1], "single" if m[2] == "f" else "half", int(m[3] or 0), int(m[4] or 0)), k


def test_nothing_in_scratch_memory_but_what_is_known():
    found = list(_found())
    if not found:
        pytest.skip("the library's code objects are compressed")
    assert {n for (n, _, _, _), _ in found} >= {"attention_rows_kernel", "attention_keys_kernel", "attention_grad_kv_kernel", "attention_grad_q_kernel", "gated_tile_kernel",
                                                "gated_rows_kernel", "gated_wide_kernel", "head_norm_rotary_kernel", "head_norm_rotary_grad_kernel"}
    over = {key: k[".vgpr_spill_count"] for key, k in found if k[".vgpr_spill_count"] > SHORT.get(key, 0) and not (key[0].startswith("attention") and key[2] == WIDEST)}
    assert not over


def test_three_waves_a_simd_for_the_gradients_of_short_heads():
    """heads of up to 64 halves or 32 floats: a third of the 512 registers, in granules of 8"""
    found = [(key, k) for key, k in _found() if key[0] == "attention_grad_kv_kernel" and key[2] * (2 if key[1] == "half" else 4) <= 128]
    if not found:
        pytest.skip("the library's code objects are compressed")
    assert not {key: k[".vgpr_count"] for key, k in found if k[".vgpr_count"] > 168}
