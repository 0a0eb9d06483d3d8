"""Which kernel the library runs for a product of a 16-bit Linear layer, and in how many slices of its inner
size (its own choice, asked without a GPU)."""
import ctypes

from cudeep_amd import _lib as L


def linear16_kernel(kind, M, N, K, aligned=True):
    """Of the product M x N x K of `kind`: "forward", "input" or "weight"."""
    f = L.lib().cdxi_linear16_kernel
    f.restype = ctypes.c_char_p
    f.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    slices = ctypes.c_int()
    name = f(("forward", "input", "weight").index(kind), M, N, K, int(aligned), ctypes.byref(slices))
    return name.decode(), slices.value
