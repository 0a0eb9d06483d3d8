"""Which kernel the library runs for an 8-bit product or weight gradient (its own choice, asked without
a GPU)."""
import ctypes

from cudeep_amd import _lib as L

_CODES = {"f32": L.DTYPE_F32, "f16": L.DTYPE_F16, "bf16": L.DTYPE_BF16}


def gemm8_kernel(M, N, K, dtype="bf16", aligned=True, from_x=False):
    """Of gemm8, or of linear8 (from_x), with results of `dtype`."""
    f = L.lib().cdxi_gemm8_kernel
    f.restype, f.argtypes = ctypes.c_char_p, [ctypes.c_int] * 2 + [ctypes.c_int64] * 3 + [ctypes.c_int]
    return f(int(from_x), _CODES[dtype], M, N, K, int(aligned)).decode()


def wgrad8_plan(M, N, K):
    """(side of the tiles, slices of the batch)."""
    f = L.lib().cdxi_wgrad8_plan
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_int64] * 3
    return divmod(f(M, N, K), 1000)
