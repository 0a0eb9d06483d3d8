"""The kernels that products of a 16-bit Linear layer run (no GPU needed): both sides of each line, and
sizes that no launch holds."""
import ctypes

import pytest

from cudeep_amd import _lib as L
from tests.routes16 import linear16_kernel

P, C = ctypes.c_void_p(0x100000), ctypes.c_void_p(1 << 60)   # never dereferenced
BF16 = 3


@pytest.mark.parametrize("M,N,K,aligned,want", [
    (1, 4096, 4096, True, "direct"), (1, 4096, 4104, True, "ring 64"), (16, 4112, 4096, True, "ring 64"),
    (32, 4096, 2048, True, "direct"), (33, 4096, 2048, True, "ring 64"), (128, 1024, 1024, True, "direct"),
    (129, 1024, 1024, True, "ring 64"), (64, 4096, 63, True, "direct"), (64, 4096, 2048, False, "direct"),
    (64, 4096, 2049, False, "any"), (1, 4096, 4001, False, "direct"),
    (2, 4096, 4001, False, "any"), (64, 4097, 333, False, "any"), (65, 4096, 333, False, "any"),
    (65, 17920, 333, False, "any 128"), (64, 17920, 333, False, "any"), (65, 17792, 333, False, "any"),
    (640, 1664, 8193, False, "any 128"), (640, 1664, 4001, False, "any"), (300, 700, 100001, False, "any 128"),
    (16, 32768, 64, True, "ring 128"), (16, 40000, 64, True, "tile 128"), (1, 128256, 4096, True, "tile 128"),
    (128, 128256, 4096, True, "tile 128"), (129, 128256, 4096, True, "turns"),
    (1024, 1024, 1280, True, "ring 64"), (1025, 1024, 1280, True, "tall"), (1024, 2048, 1280, True, "tall"),
    (1025, 2048, 1280, True, "ring 128"), (2048, 1024, 4096, True, "tall"), (1152, 1152, 8192, True, "ring 128"),
    (1152, 1152, 8128, True, "tall"), (1400, 1600, 1280, True, "ring 128"),
    (1024, 1024, 8192, True, "ring 128"), (1024, 1024, 8128, True, "ring 64"), (2048, 2048, 2048, True, "ring 128"),
    (2048, 2176, 2048, True, "tile 128"), (2048, 2176, 63, True, "any 128"), (3584, 3584, 512, True, "tile 128"),
    (2560, 5120, 512, True, "turns"), (512, 512, 65536, True, "ring 128"), (1024, 1024, 65536, True, "turns"),
    (256, 256, 16384, True, "ring 64"),
])
def test_forward(M, N, K, aligned, want):
    assert linear16_kernel("forward", M, N, K, aligned)[0] == want
    if want != "direct":
        for kind in ("input", "weight"):
            assert linear16_kernel(kind, M, N, K, aligned)[0] == want


@pytest.mark.parametrize("M,N,K,aligned,slices", [
    (64, 4096, 4096, True, 4), (1024, 1024, 4096, True, 1), (256, 256, 16384, True, 8), (256, 784, 8192, True, 4),
    (1024, 1024, 65536, True, 16), (512, 512, 65536, True, 16), (256, 784, 8192, False, 9), (16, 640, 6575, False, 15), (1336, 1440, 8026, False, 3), (256, 512, 65536, True, 16),
    (300, 1000, 200, True, 1),
])
def test_slices(M, N, K, aligned, slices):
    assert linear16_kernel("weight", M, N, K, aligned)[1] == slices
    size = L.lib().cdx_linear16_backward_workspace_size(K, M, N, 0)
    assert size >= (slices * (M * N + M) * 4 if slices > 1 else 0)


def test_products_that_no_launch_holds():
    """2^23 tiles and more, of 64 x 64 and of 128 x 128."""
    for M, N in ((1 << 20, 1 << 20), (1, 1 << 30), (1 << 18, 1 << 22)):
        st = L.lib().cdx_linear16(M, N, 16, P, 16, P, 16, None, BF16, None, N, C, N, None, N, 0, BF16, None, 0, None)
        assert st == L.CDX_ERR_UNSUPPORTED and b"tiles" in L.lib().cdx_last_error(), (M, N)


def test_queries_of_sizes_that_nothing_has():
    """Products beyond 2^58 elements: the queries answer 0 (the call itself refuses them)."""
    for M, N, K in ((1 << 40, 1 << 40, 64), (1 << 40, 64, 1 << 40), (64, 1 << 40, 1 << 40), (1 << 36, 1 << 36, 1 << 36)):
        assert L.lib().cdx_linear16_workspace_size(M, N, K) == 0
        assert L.lib().cdx_linear16_backward_workspace_size(M, N, K, 2) == 0
        assert L.lib().cdx_linear16(M, N, K, P, K, P, K, None, BF16, None, N, C, N, None, N, 0, BF16, None, 0,
                                    None) == L.CDX_ERR_INVALID_ARG


def test_logits_parts():
    f = L.lib().cdxi_logits_parts
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    for op, rows, vocab, top, want in [(0, 1, 65536, 5, 1), (0, 1, 131072, 5, 8), (0, 1, 131072, 64, 8),
                                       (0, 1, 400000, 64, 16), (0, 127, 131072, 0, 4), (0, 128, 131072, 0, 1),
                                       (1, 16, 65535, 0, 1), (1, 16, 65536, 0, 4), (1, 16, 131072, 0, 8), (1, 128, 131072, 0, 1)]:
        assert f(op, rows, vocab, top) == want, (op, rows, vocab, top)


def test_rows_that_no_launch_holds():
    n = 1 << 24
    assert L.lib().cdx_token_logprobs(P, 8, n, 8, 0, 1.0, P, P, P, None, 0, None, None, None, 0, None) == L.CDX_ERR_UNSUPPORTED
    assert L.lib().cdx_distill_loss(P, 8, n, 8, 0, 1.0, P, 1, 8, P, 1, 0, 1, P, None, None, 0, None, 0, None) == L.CDX_ERR_UNSUPPORTED
    # 2^24 workgroups of the gradient
    assert L.lib().cdx_token_logprobs_backward(P, C, 4096, n, 4096, 0, 1.0, P, P, None, None, C, 4096, None) == L.CDX_ERR_UNSUPPORTED


def test_workspaces_begin_on_16_bytes():
    odd = ctypes.c_void_p(0x100008)
    assert L.lib().cdx_linear16(4, 8, 16, P, 16, P, 16, None, BF16, None, 8, C, 8, None, 8, 0, BF16, odd, 1 << 20,
                                None) == L.CDX_ERR_INVALID_ARG
    assert L.lib().cdx_token_logprobs(P, 8, 1, 8, 0, 1.0, P, P, P, None, 0, None, None, odd, 64, None) == L.CDX_ERR_INVALID_ARG
    assert L.lib().cdx_distill_loss(P, 8, 1, 8, 0, 1.0, P, 1, 8, P, 1, 0, 1, P, None, None, 0, odd, 64, None) == L.CDX_ERR_INVALID_ARG
