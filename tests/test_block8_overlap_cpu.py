"""Results that overlap their inputs: refused on the host, before any launch, unless an operator takes
each row in its place.  (few rows of cdx_linear_e4m3 are read by every workgroup while others write.)"""
import ctypes

import pytest

from cudeep_amd import _lib as L

BASE = 0x10000   # never dereferenced: validation fails first
F32, F16, BF16, E8 = 0, 2, 3, 4
P = ctypes.c_void_p(0x9000000)


def _refused(name, *args):
    status = getattr(L.lib(), name)(*args)
    return status == L.CDX_ERR_INVALID_ARG and b"overlap" in L.lib().cdx_last_error()


# offsets in bytes of the result from the input, and leading dimensions: [8, 64] matrices
SHIFTS = [(2, 64, 64), (-2, 64, 64), (128, 64, 64), (-128, 64, 64), (0, 64, 65), (128, 96, 96),
          (66, 96, 96), (-66, 96, 96), (7 * 128 + 126, 64, 64), (-(7 * 128 + 126), 64, 64)]


@pytest.mark.parametrize("shift,ldx,ldy", SHIFTS)
def test_rows_out_of_place(shift, ldx, ldy):
    x, y = ctypes.c_void_p(BASE), ctypes.c_void_p(BASE + shift)
    assert _refused("cdx_layer_norm_forward", x, ldx, None, None, y, ldy, None, None, 8, 64, 1e-5,
                    BF16, BF16, None)
    back = [P, 64, P, 64, None, P, P, y, ldy, None, None, 8, 64, BF16, BF16, None, 0, None]
    for at in (0, 2):
        args = list(back)
        args[at], args[at + 1] = x, ldx
        assert _refused("cdx_layer_norm_backward", *args)
    assert _refused("cdx_activation_forward_e4m3", x, ldx, y, ldy, P, 64, P, 1, E8, 8, 64, BF16, 2,
                    0.0, None)
    assert _refused("cdx_activation_backward_e4m3", x, ldx, P, 64, P, 1, E8, y, ldy, 8, 64, BF16, 2,
                    0.0, None)


@pytest.mark.parametrize("shift,ldx,ldy", SHIFTS + [(0, 64, 64), (0, 96, 96)])
def test_products(shift, ldx, ldy):
    x, c = ctypes.c_void_p(BASE), ctypes.c_void_p(BASE + shift)
    assert _refused("cdx_linear_e4m3", 8, 64, 64, x, ldx, BF16, P, 64, P, 1, E8, c, ldy, BF16, None, 0,
                    None, 0, None)
    # one row: the bytes themselves
    one = -126 if shift < 0 else min(shift, 126)
    assert _refused("cdx_linear_e4m3", 1, 64, 64, x, ldx, BF16, P, 64, P, 1, E8,
                    ctypes.c_void_p(BASE + one), ldy, BF16, None, 0, None, 0, None)
