"""The example of a transformer block on the host layer: trained, then served from a cache of keys and values."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu
EXAMPLE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deep8_amd", "host", "deep8_transformer_block")


def test_block_learns_and_serves_what_it_learnt():
    out = subprocess.run([EXAMPLE, "60"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0 and out.stdout.endswith("OK\n"), out.stdout + out.stderr
