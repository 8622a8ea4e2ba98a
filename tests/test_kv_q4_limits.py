"""Arguments at the ends of their types, checked before any device call."""
import ctypes as C
import subprocess
import sys

import numpy as np
import pytest

from alpaca_amd import _lib as L

CTX = C.create_string_buffer(64)  # stands for a context in calls that are refused before they use it


@pytest.mark.parametrize("kv", [L.KV_F16, L.KV_F32, L.KV_Q4_0])
def test_op_attention_past_the_last_position(kv):
    x = np.zeros((1, 1, 32), np.float32)
    p = x.ctypes.data_as(L.fp)
    for start, capacity in ((1, 1), (2**31 - 1, 1), (0, -2**31)):  # (the end is past 31 bits, or its distance)
        rc = L.lib().ahip_op_attention(C.addressof(CTX), p, 1, 1, 32, p, p, capacity, 1, start, kv, L.GEMM_EXACT, p)
        assert rc == L.INVALID_ARGUMENT and b"shapes" in L.lib().ahip_last_error()


def test_session_bytes_of_the_largest_capacities():
    """A size query walks the call lengths that need a workspace, not all up to the capacity (200 s)."""
    code = """
from alpaca_amd import synth
from alpaca_amd.model import HIPLlamaModel
for spec in (synth.C1, synth.C5, synth.TINY):
    c = spec.config
    a, b, d = (HIPLlamaModel.session_byte_count(c, 1 << 30, n << 28, "q4_0") for n in (1, 2, 3))
    assert b - a == d - b > 0  # what a token of the batch takes
    cache = 2 * c.layer_count * (1 << 30) * c.kv_width * 18 // 32
    assert a > cache + 4 * (1 << 28) * c.hidden_size
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=60)
