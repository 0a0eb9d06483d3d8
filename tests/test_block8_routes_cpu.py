"""The kernels that 8-bit products and weight gradients run (no GPU needed): both sides of each line."""
import pytest

from tests.routes8 import gemm8_kernel, wgrad8_plan


@pytest.mark.parametrize("M,N,K,aligned,want", [
    (1, 4096, 4096, True, "direct"), (32, 4096, 4096, True, "direct"), (33, 4096, 4096, True, "ring"),
    (64, 4096, 2047, True, "direct"), (64, 4096, 2048, True, "ring"), (64, 4096, 4096, False, "direct"),
    (65, 4096, 4096, False, "direct"), (1024, 1024, 1024, True, "ring"), (1024, 896, 1024, True, "direct"),
    (1024, 1024, 1024, False, "any"), (1024, 1024, 127, True, "any"), (1024, 1024, 128, True, "ring"),
    (512, 4096, 4096, True, "ring"), (576, 4096, 4096, True, "tile 128"),
    (2560, 5120, 1024, True, "tile 256"), (2304, 5120, 1024, True, "tile 128"),
    (2560, 5120, 1024, False, "any"), (5, 5, 0, True, "empty"),
])
def test_products(M, N, K, aligned, want):
    for dtype in ("bf16", "f16"):
        assert gemm8_kernel(M, N, K, dtype, aligned) == want
    # results of 32 bits have no 256-wide tiles
    assert gemm8_kernel(M, N, K, "f32", aligned) == want.replace("256", "128")


@pytest.mark.parametrize("M,K,inside", [(1, 4096, True), (1, 4097, False), (16, 4096, True), (17, 4096, False),
                                        (17, 2891, True), (17, 2892, False), (64, 768, True), (64, 769, False),
                                        (65, 100, False)])
def test_input_quantised_inside(M, K, inside):
    got = gemm8_kernel(M, 1000, K, from_x=True)
    assert (got == "direct, quantises") == inside
    # the kernel that the codes alone would run, so that the bits are the same
    if inside:
        assert gemm8_kernel(M, 1000, K) == "direct"
    else:
        assert got == gemm8_kernel(M, 1000, K)


@pytest.mark.parametrize("M,N,K,side,slices", [
    (64, 250, 333, 64, 1), (2100, 256, 784, 64, 7), (3510, 256, 784, 64, 8), (3511, 256, 784, 128, 11),
    (1030, 770, 900, 128, 4), (200, 2050, 2050, 128, 1), (170, 2050, 2050, 64, 1),
    (6000, 250, 790, 128, 19), (4100, 2050, 1800, 256, 3), (3640, 2050, 1800, 128, 2),
    (100, 4100, 4000, 256, 1), (100, 3840, 3900, 128, 1), (300, 40, 0, 64, 1),
])
def test_weight_gradients(M, N, K, side, slices):
    assert wgrad8_plan(M, N, K) == (side, slices)
