"""Sums of 8-bit products that cancel.  Results of float32 come from sums that hold 24 bits: beside
products of 2^16 and -2^16 one of 3 counts.  Results of 16 bits come from the 8-bit matrix
instruction, which adds eight products on a grid 2^-13 below the power of two of the largest: beside
2^16 every multiple of 8 counts whole."""
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _operands(M, N, K, small, scale, shift):
    """In every eight columns 256 * 256 - 256 * 256 + small n, n = 1 or -1 by the row of B; with shift
    the rows of the codes begin at odd bytes."""
    import torch
    from cudeep_amd import ops
    a = torch.tensor([256.0, small, 0, 256.0, 0, 0, 0, 0], device="cuda").repeat(K // 8).expand(M, K)
    b = torch.tensor([256.0, 1.0, 0, -256.0, 0, 0, 0, 0], device="cuda").repeat(K // 8).repeat(N, 1)
    b[1::2, 1::8] = -1.0

    def block(v, tiles, tile_rows):
        q = torch.zeros((v.shape[0], K + shift), device="cuda").to(torch.float8_e4m3fn)
        q[:, shift:] = v.to(torch.float8_e4m3fn)
        s = torch.ones((tiles, -(-K // 128)), device="cuda")
        return ops.Block8(q[:, shift:], s if scale == "f32" else s.to(torch.float8_e8m0fnu), tile_rows)

    want = torch.full((M, N), small * (K // 8), device="cuda")
    want[:, 1::2] *= -1
    return block(a, M, 1), block(b, -(-N // 128), 128), want


# sizes of every kernel: straight from global memory, the ring, 128- and 256-wide tiles, rows at any byte
@pytest.mark.parametrize("dtype,small", [("float32", 3.0), ("float16", 24.0), ("bfloat16", 24.0)])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("size", [(1, 40, 1000, 0), (20, 100, 512, 0), (50, 33, 640, 0), (60, 200, 2048, 0),
                                  (520, 2000, 640, 0), (1100, 2300, 512, 0), (3590, 3601, 304, 0),
                                  (1100, 1300, 520, 1)])
def test_sums_that_cancel(size, scale, dtype, small):
    import torch
    from cudeep_amd import ops
    M, N, K, shift = size
    a, b, want = _operands(M, N, K, small, scale, shift)
    say("gemm8 sums that cancel", size, scale, dtype)
    dt = getattr(torch, dtype)
    assert torch.equal(ops.gemm8(a, b, dtype=dt), want.to(dt))


@pytest.mark.parametrize("size", [(1, 40, 1000), (40, 100, 1000), (300, 260, 512), (1100, 2300, 512)])
def test_linear_sums_that_cancel(size):
    """From 16-bit rows, with float32 and with 16-bit results."""
    import torch
    from cudeep_amd import ops
    M, N, K = size
    say("linear8 sums that cancel", size)
    for small, dt in ((3.0, torch.float32), (24.0, torch.float16)):
        a, b, want = _operands(M, N, K, small, "e8m0", 0)
        x = ops.dequantize8(a, torch.float16)
        assert torch.equal(ops.linear8(x, b, dtype=dt), want.to(dt))
