"""Products and weight gradients of more output tiles than a launch holds are refused on the host."""
import ctypes

from cudeep_amd import _lib as L

P, C = ctypes.c_void_p(0x1000), ctypes.c_void_p(1 << 60)   # never dereferenced
F32, BF16, E8 = 0, 3, 4


def _unsupported(name, *args):
    return getattr(L.lib(), name)(*args) == L.CDX_ERR_UNSUPPORTED and b"tiles" in L.lib().cdx_last_error()


def test_products():
    # straight from global memory, 16 columns and 512 threads a workgroup; 64 x 64 tiles of 256 threads
    for M, N, K in ((1, (1 << 27) + 16, 16), (60, (1 << 27) + 16, 16), (1 << 18, 1 << 18, 16)):
        assert _unsupported("cdx_gemm_e4m3", M, N, K, P, K, P, 1, E8, P, K, P, 1, E8, C, N, BF16, None, 0,
                            None, 0, None)
    assert _unsupported("cdx_linear_e4m3", 1, 1 << 27, 16, P, 16, BF16, P, 16, P, 1, E8, C, 1 << 27, BF16,
                        None, 0, None, 0, None)


def test_weight_gradients():
    n = 1 << 20
    assert _unsupported("cdx_linear_weight_grad_e4m3", P, n, F32, P, n, P, n // 128, C, P, 64, n, n, None,
                        0, None)
