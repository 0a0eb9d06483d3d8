"""What a call of the 16-bit Linear layer needs of its workspace goes by its own operands (no GPU needed): never more
than the sizes' query answers, nothing where its products run in one slice, and less is refused."""
import ctypes
import random

from cudeep_amd import _lib as L
from tests.routes16 import linear16_kernel

BF16 = 3


def _at(k):   # never dereferenced: the calls are refused
    return ctypes.c_void_p(0x100000 + 0x40000000 * k)


def _forward(M, N, K, odd=0):
    x = ctypes.c_void_p(_at(0).value + 2 * odd)
    return L.lib().cdx_linear16_call_workspace_size(M, N, K, x, K + odd, _at(1), K)


def _backward(M, N, K, epilogue, input=1, params=1, bias=1, odd=0):
    return L.lib().cdx_linear16_backward_call_workspace_size(M, N, K, _at(0), N + odd, _at(1), K, _at(2), K, epilogue, input,
                                                             params, bias)


def test_one_launch_needs_nothing():
    for M, N, K in ((48, 200, 4096), (2, 4096, 4096), (16, 4096, 4096)):
        assert linear16_kernel("forward", M, N, K) == ("direct", 1)
        assert L.lib().cdx_linear16_workspace_size(M, N, K) > 0       # operands of another alignment would be sliced
        assert _forward(M, N, K) == 0 and _forward(M, N, K, odd=1) == L.lib().cdx_linear16_workspace_size(M, N, K)


def test_a_call_needs_no_more_than_its_sizes():
    rng = random.Random(0)
    for _ in range(3000):
        M, N, K = (int(2 ** rng.uniform(0, 14)) // rng.choice([1, 8]) * rng.choice([1, 8]) for _ in range(3))
        odd, act = rng.choice([0, 1, 8]), rng.choice([0, 1, 2, 3, 4])
        assert _forward(M, N, K, odd) <= L.lib().cdx_linear16_workspace_size(M, N, K)
        most = L.lib().cdx_linear16_backward_workspace_size(M, N, K, act)
        whole = _backward(M, N, K, act, odd=odd)
        assert whole <= most
        for some in ((1, 0, 0), (0, 1, 0), (0, 1, 1), (1, 1, 0)):
            assert _backward(M, N, K, act, *some, odd=odd) <= whole
        assert _backward(M, N, K, act, 0, 0, 0) == 0


def test_the_parts_add_up():
    M, N, K = 8192, 256, 784        # weight gradient in slices, input gradient in one
    slices = linear16_kernel("weight", N, K, M)[1]
    assert slices > 1 and linear16_kernel("input", M, K, N)[1] == 1
    assert _backward(M, N, K, 0, 1, 0, 0) == 0
    assert _backward(M, N, K, 0, 0, 1, 0) == slices * N * K * 4
    assert _backward(M, N, K, 0) == slices * (N * K + N) * 4          # with the bias's column sums
    assert _backward(M, N, K, 1) == M * N * 2 + slices * (N * K + N) * 4
    with_sums, without = _backward(M, N, K, 2), _backward(M, N, K, 2, bias=0)
    assert without == M * N * 2 + slices * N * K * 4 < with_sums      # the slopes' sums


def test_less_is_refused():
    M, N, K, ws = 64, 8192, 4096, _at(9)
    need = _forward(M, N, K)
    assert need > 0
    st = L.lib().cdx_linear16(M, N, K, _at(0), K, _at(1), K, None, BF16, None, N, _at(2), N, None, N, 0, BF16, ws, need - 1,
                              None)
    assert st == L.CDX_ERR_WORKSPACE
    for act in (0, 1, 2):
        M, N, K = 8192, 256, 784
        need = _backward(M, N, K, act)
        st = L.lib().cdx_linear16_backward(M, N, K, _at(0), N, _at(1), K, _at(2), K, _at(3), N, act, _at(4), K, _at(5), _at(6),
                                           BF16, BF16, ws, need - 1, None)
        assert st == L.CDX_ERR_WORKSPACE
