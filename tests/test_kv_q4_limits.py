"""Arguments at the ends of their types, checked before any device call."""
import ctypes as C

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
