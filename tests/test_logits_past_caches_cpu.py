"""What of a gradient of logits passes the caches by (no GPU needed): both sides of each line."""
import ctypes

import pytest

from cudeep_amd import _lib as L

F32, F16, BF16 = 0, 2, 3
NOTHING, LOGITS, BOTH = 0, 1, 2


@pytest.mark.parametrize("rows,vocab,dtype,want", [
    (319, 50000, F32, NOTHING), (320, 50000, F32, BOTH), (513, 50001, F32, BOTH), (4000, 50000, F32, BOTH),
    (639, 50000, BF16, NOTHING), (640, 50000, BF16, LOGITS), (1999, 50000, BF16, LOGITS), (2000, 50000, BF16, BOTH),
    (639, 50000, F16, NOTHING), (1999, 50000, F16, LOGITS), (4096, 65536, F16, BOTH), (1, 50000, BF16, NOTHING),
])
def test_lines(rows, vocab, dtype, want):
    f = L.lib().cdxi_logits_past_caches
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    assert f(rows, vocab, dtype) == want
