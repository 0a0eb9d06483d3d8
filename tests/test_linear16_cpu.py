"""The 16-bit Linear layer's C entry points refuse bad arguments before any launch, their size queries
answer without a GPU, and the wrappers refuse what is not on one."""
import ctypes

import pytest

from cudeep_amd import _lib as L

P = ctypes.c_void_p(0x100000)   # never dereferenced: validation fails first
F32, F64, F16, BF16 = 0, 1, 2, 3


def _at(k):
    return ctypes.c_void_p(0x100000 + 0x100000 * k)


def _status(name, *args):
    return getattr(L.lib(), name)(*args)


def _bad(name, good, changes):
    """Every change {position: value} of the good arguments is refused."""
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert _status(name, *args) == L.CDX_ERR_INVALID_ARG, (name, at, value)
        assert name.encode() in L.lib().cdx_last_error()


# M, N, K, x, ldx, w, ldw, bias, bias_dtype, residual, ldr, y, ldy, z, ldz, epilogue, dtype, ws, bytes, stream
FORWARD = [40, 8, 200, _at(0), 200, _at(1), 200, _at(2), F32, _at(3), 8, _at(4), 8, _at(5), 8, 2, BF16, None, 0, None]
# M, N, K, dy, ldg, x, ldx, w, ldw, z, ldz, epilogue, dx, lddx, dw, db, dtype, param_dtype, ws, bytes, stream
BACKWARD = [40, 8, 200, _at(0), 8, _at(1), 200, _at(2), 200, _at(3), 8, 2, _at(4), 200, _at(5), _at(6), BF16, BF16,
            _at(7), 1 << 30, None]


def test_forward_arguments():
    _bad("cdx_linear16", FORWARD, [
        (0, -1), (1, -1), (2, -1), (0, 1 << 41), (3, None), (4, 199), (5, None), (6, 199), (8, F64), (8, F16),
        (10, 7), (11, None), (12, 7), (14, 7), (15, 5), (15, 8), (15, -1), (16, F32), (16, F64)])
    # results over what is still read, or over each other
    _bad("cdx_linear16", FORWARD, [(11, _at(0)), (11, _at(1)), (11, _at(2)), (11, _at(5)), (13, _at(0)), (13, _at(1)),
                                   (13, _at(2)), (13, _at(3)), (11, ctypes.c_void_p(_at(3).value + 2))])
    for empty in (0, 1):
        args = [0 if i == empty else v for i, v in enumerate(FORWARD)]
        assert _status("cdx_linear16", *args) == L.CDX_OK


def test_backward_arguments():
    _bad("cdx_linear16_backward", BACKWARD, [
        (0, -1), (1, -1), (2, -1), (3, None), (4, 7), (5, None), (6, 199), (7, None), (8, 199), (9, None), (10, 7),
        (11, 5), (13, 199), (14, None), (16, F32), (17, F16), (17, F64)])
    _bad("cdx_linear16_backward", BACKWARD, [(at, _at(k)) for at, own in ((12, 4), (14, 5), (15, 6))
                                             for k in range(7) if k != own])
    small = list(BACKWARD)
    small[19] = 4
    assert _status("cdx_linear16_backward", *small) == L.CDX_ERR_WORKSPACE
    nothing = list(BACKWARD)
    nothing[12] = nothing[14] = nothing[15] = None
    assert _status("cdx_linear16_backward", *nothing) == L.CDX_OK


def test_workspace_sizes():
    assert _status("cdx_linear16_workspace_size", 8192, 4096, 4096) == 0
    assert _status("cdx_linear16_workspace_size", -1, 8, 8) == 0
    # with an activation, dz
    assert _status("cdx_linear16_backward_workspace_size", 40, 8, 200, 2) >= 40 * 8 * 2
    assert _status("cdx_linear16_backward_workspace_size", 0, 8, 200, 0) == 0


def test_wrappers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from cudeep_amd import ops
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    for f in (lambda: ops.linear16(x, w), lambda: ops.linear16_backward(x, x, w), lambda: ops.linear16([1], w)):
        with pytest.raises((ValueError, TypeError)):
            f()


def test_a_layer_without_inputs_takes_the_kernel_that_reads_none():
    from tests.routes16 import linear16_kernel
    for M, K in ((24, 130), (4096, 8192), (8, 64)):
        assert linear16_kernel("weight", M, 0, K) == ("any", 1)
