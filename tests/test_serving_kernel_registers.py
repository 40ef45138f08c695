"""Registers of the kernels of the norm of rows, the 8-bit products and the 8-bit cache, read from the code objects of the built library: what lies in
scratch memory, and how many waves a SIMD has room for."""
import re

import pytest

from deep8_amd import capi
from test_kernel_registers import _code_objects, _kernels

NAMES = ("layer_norm_kernel", "layer_norm_grad_kernel", "layer_norm_long_kernel", "layer_norm_grad_long_kernel", "layer_norm_sums_kernel", "quantize_rows_kernel",
         "quantize_long_rows_kernel", "cache_append_kernel", "cache_read_kernel", "attention_cache_kernel", "attention_cache_join_kernel")
# gradients of rows of more than 8192 elements, 16 a thread of 1024: half, with what moves a row's last piece down; single either way
SHORT = {("layer_norm_grad_kernel", "DF16_Li8ELi1024ELi16ELb1E"): 20, ("layer_norm_grad_kernel", "fLi4ELi1024ELi16ELb0E"): 10, ("layer_norm_grad_kernel", "fLi4ELi1024ELi16ELb1E"): 14}

def _found():
    with open(capi.LIB_PATH, "rb") as f:
        blob = f.read()
    for at in _code_objects(blob):
        for k in _kernels(blob, at):
            m = re.search(r"\d(" + "|".join(NAMES) + r")(?:I(\w*?)EEv)?", k[".name"])
            if m or "int8" in k[".name"] or "Int8" in k[".name"]:
                yield (m[1], m[2] or "") if m else ("int8", k[".name"]), k


@pytest.fixture(scope="module")
def found():
    kernels = list(_found())
    if not kernels:
        pytest.skip("the library's code objects are compressed")
    return kernels


def test_nothing_in_scratch_memory_but_what_is_known(found):
    assert {n for (n, _), _ in found} == set(NAMES) | {"int8"}
    assert not {key: k[".vgpr_spill_count"] for key, k in found if k[".vgpr_spill_count"] > SHORT.get(key, 0)}


def test_waves_a_simd(found):
    """what the launches count on: attention in half over heads of up to 128 elements, two workgroups of eight waves a compute unit (128 of a SIMD's 512
    registers a wave) where they share pages and two of four waves (256) where they do not; norm gradients of 8 elements a thread, two of eight (128)"""
    held = {key: k[".vgpr_count"] for key, k in found}
    rows = [n for (name, args), n in held.items() if name == "attention_cache_kernel" and re.match(r"DF16_Li[12]ELb1", args)]
    keys = [n for (name, args), n in held.items() if name == "attention_cache_kernel" and re.match(r"(DF16_|f)Li[12]ELb0", args)]
    grads = [n for (name, args), n in held.items() if name == "layer_norm_grad_kernel" and "ELi8ELb" in args]
    assert len(rows) == 2 and len(keys) == 4 and len(grads) >= 8
    assert max(rows) <= 128 and max(keys) <= 256 and max(grads) <= 128
