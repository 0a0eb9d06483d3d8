"""Every kernel of the 8-bit products with bias and activation, with scales of two kinds, NaN, the
scale bytes' ends and rows at any byte; linear8 by each of them.  Which kernel runs is asserted.

Bounds as in test_gpu_block8.py: products are exact and K + 8 additions round by 2^-24 of the sum of
magnitudes each; results of 16 bits lose 2^-10 of the largest of each eight products besides."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.routes8 import gemm8_kernel
from tests.test_gpu_block8 import U, _dtype, _half_ulp, _normal, _operands, _values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _double(b):
    import torch
    return torch.from_numpy(_values(b)).cuda()


def _check(got, a, b, bias=None, act="none"):
    """got against act(A B^T + bias) of float64 matrices on the device."""
    import torch
    K = a.shape[1]
    exact = a @ b.t().contiguous()
    mag = a.abs() @ b.abs().t().contiguous()
    if bias is not None:
        exact, mag = exact + bias.double(), mag + bias.double().abs()
    bound = (K + 8) * U * mag
    if got.dtype != torch.float32:
        af, bf = (torch.nn.functional.pad(t.abs(), (0, -K % 8)) for t in (a, b))
        for k in range(0, K, 8):
            bound += 2.0 ** -10 * (af[:, None, k:k + 8] * bf[None, :, k:k + 8]).amax(-1)
    if act == "relu":
        exact = exact.clamp_min(0)
    elif act != "none":
        # slopes of at most 1.13, and a few roundings of the function itself
        bound = 1.13 * bound + 16 * U * (exact.abs() + 1)
        u = 2 * 0.7978845608 * (exact + 0.044715 * exact ** 3) if act == "gelu" else exact
        exact = (1.0 if act == "sigmoid" else exact) / (1 + torch.exp(-u))
    bound = bound + _half_ulp(got.dtype) * exact.abs() + 2.0 ** -25
    over = ((got.double() - exact).abs() - bound).max().item()
    assert over <= 0, over


# ragged in both directions and in K
KERNELS = {"direct": (61, 1003, 645), "ring": (515, 2009, 645), "tile 128": (1101, 2303, 517),
           "tile 256": (3590, 3601, 300)}


def _kernel(name, dtype):
    return name.replace("256", "128") if dtype == "f32" else name


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("kernel", list(KERNELS))
def test_bias_and_activation(kernel, act, dtype):
    from cudeep_amd import _lib as L
    from cudeep_amd import ops
    M, N, K = KERNELS[kernel]
    assert gemm8_kernel(M, N, K, dtype) == _kernel(kernel, dtype)
    epi = {"none": L.EPI_NONE, "relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU,
           "sigmoid": L.EPI_SIGMOID}[act]
    a, b = _operands(M, N, K, "f32" if act in ("relu", "silu") else "e8m0", 3)
    bias = _normal((1, N), 9)[0]
    say("gemm8 bias and activation", kernel, act, dtype)
    got = ops.gemm8(a, b, bias=bias, epilogue=epi, dtype=_dtype(dtype))
    _check(got, _double(a), _double(b), bias, act)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("kernel,size", [("direct, quantises", (61, 303, 700)), ("direct", (30, 303, 4001))]
                         + [(k, s) for k, s in KERNELS.items() if k != "direct"])
def test_linear(kernel, size, scale, dtype):
    """linear8(x) is gemm8(quantize8(x)) bit for bit, also of rows inside a wider matrix."""
    import torch
    from cudeep_amd import _lib as L
    from cudeep_amd import ops
    M, N, K = size
    assert gemm8_kernel(M, N, K, dtype, from_x=True) == _kernel(kernel, dtype)
    x = _normal((M, K), 5).to(_dtype(dtype))
    b = _operands(1, N, K, scale, 6)[1]
    bias = _normal((1, N), 7)[0]
    say("linear8", kernel, scale, dtype)
    got = ops.linear8(x, b, bias, epilogue=L.EPI_GELU)
    a = ops.quantize8(x, scale_dtype=_dtype(scale))
    assert torch.equal(got, ops.gemm8(a, b, bias=bias, epilogue=L.EPI_GELU, dtype=x.dtype))
    _check(got, _double(a), _double(b), bias, "gelu")
    wide = torch.full((M, K + 9), float("nan"), device="cuda", dtype=x.dtype)
    wide[:, 3:3 + K] = x
    out = torch.full((M, N + 7), 5.0, device="cuda", dtype=x.dtype)
    assert torch.equal(ops.linear8(wide[:, 3:3 + K], b, bias, epilogue=L.EPI_GELU, out=out[:, 3:3 + N]), got)
    assert (out[:, :3] == 5).all() and (out[:, 3 + N:] == 5).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kinds", [("e8m0", "f32"), ("f32", "e8m0")])
@pytest.mark.parametrize("kernel", list(KERNELS))
def test_scales_of_two_kinds(kernel, kinds, dtype):
    from cudeep_amd import ops
    M, N, K = KERNELS[kernel]
    a, b = _operands(M, N, K, kinds[0], 13)[0], _operands(M, N, K, kinds[1], 13)[1]
    say("gemm8 scales of two kinds", kernel, kinds, dtype)
    _check(ops.gemm8(a, b, dtype=_dtype(dtype)), _double(a), _double(b))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("shift", [1, 4])
def test_rows_at_any_byte(shift, scale, dtype):
    """The kernel for unaligned rows; NaN codes lie around the views."""
    import torch
    from cudeep_amd import _lib as L
    from cudeep_amd import ops
    M, N, K = 1101, 1303, 517
    assert gemm8_kernel(M, N, K, dtype, aligned=False) == "any"
    a, b = _operands(M, N, K, scale, 8)
    bias = _normal((1, N), 9)[0]

    def inside(t, pad):
        wide = torch.full((t.shape[0], t.shape[1] + pad + shift), 0x7f, dtype=torch.uint8, device="cuda")
        wide[:, shift:shift + t.shape[1]] = t.view(torch.uint8)
        return wide.view(t.dtype)[:, shift:shift + t.shape[1]]

    a2 = ops.Block8(inside(a.q, 3), a.scale, 1)
    b2 = ops.Block8(inside(b.q, 5), b.scale, 128)
    say("gemm8 rows at any byte", shift, scale, dtype)
    got = ops.gemm8(a2, b2, bias=bias, epilogue=L.EPI_SILU, dtype=_dtype(dtype))
    _check(got, _double(a), _double(b), bias, "silu")
    # blocks of less than one whole 128
    got = ops.gemm8(ops.Block8(a2.q[:, :100], a2.scale[:, :1], 1), ops.Block8(b2.q[:, :100], b2.scale[:, :1], 128),
                    dtype=_dtype(dtype))
    _check(got, _double(a)[:, :100], _double(b)[:, :100])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("kernel", list(KERNELS))
def test_nan_and_extreme_scales(kernel, scale, dtype):
    """NaN codes and scales reach their own rows and columns alone; products of the largest and
    the smallest powers of two as scales."""
    import torch
    from cudeep_amd import ops
    M, N, K = KERNELS[kernel]
    a, b = _operands(M, N, K, "e8m0", 12)
    sa, sb = a.scale.view(torch.uint8), b.scale.view(torch.uint8)
    sa[:, 0], sb[:, 0] = 240, 20     # 2^113 * 2^-107
    sa[:, 1], sb[:, 1] = 14, 246     # 2^-113 * 2^119
    sa[:, 2], sb[:, 2] = 1, 254      # 2^-126 * 2^127
    if scale == "f32":
        a = ops.Block8(a.q, torch.exp2(sa.float() - 127), 1)
        b = ops.Block8(b.q, torch.exp2(sb.float() - 127), 128)
    say("gemm8 extreme scales", kernel, scale, dtype)
    clean = ops.gemm8(a, b, dtype=torch.float32)
    got = ops.gemm8(a, b, dtype=_dtype(dtype))
    if dtype != "f16":   # (beyond f16's range)
        _check(got, _double(a), _double(b))
    else:
        assert not got.isnan().any() and got.isfinite().all() == (clean.abs() < 65520).all()
    a.q.view(torch.uint8)[3, 131] = 0x7f
    b.q.view(torch.uint8)[N - 1, 7] = 0xff
    if scale == "f32":
        a.scale[5, 1] = float("nan")
    else:
        a.scale.view(torch.uint8)[5, 1] = 255
    bad = ops.gemm8(a, b, dtype=_dtype(dtype))
    assert bad[3].isnan().all() and bad[5].isnan().all() and bad[:, N - 1].isnan().all()
    bad[3], bad[5], bad[:, N - 1] = got[3], got[5], got[:, N - 1]
    assert torch.equal(bad, got)
    # a tile's scale: 128 columns
    if scale == "f32":
        b.scale[1, 0] = float("nan")
    else:
        b.scale.view(torch.uint8)[1, 0] = 255
    bad = ops.gemm8(a, b, dtype=_dtype(dtype))
    assert bad[:, 128:256].isnan().all()
    bad[3], bad[5], bad[:, N - 1], bad[:, 128:256] = got[3], got[5], got[:, N - 1], got[:, 128:256]
    assert torch.equal(bad, got)


def test_rows_of_more_blocks_than_31_bits_hold():
    """Quantising and restoring 2^31 + 5 rows of one column, and rows that a grid walks twice."""
    import torch
    from cudeep_amd import ops
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    for rows, cols in (((1 << 31) + 5, 1), ((1 << 24) + 37, 100)):
        x = torch.zeros((rows, cols), device="cuda", dtype=torch.bfloat16)
        tail = _normal((7, cols), 3).to(torch.bfloat16)
        x[-7:] = tail
        say("quantize8", rows, cols)
        b = ops.quantize8(x)
        want = ops.quantize8(tail)
        assert torch.equal(b.q[-7:].view(torch.uint8), want.q.view(torch.uint8))
        assert torch.equal(b.scale[-7:].view(torch.uint8), want.scale.view(torch.uint8))
        assert (b.scale[:-7].view(torch.uint8) == 127).all()
        del x
        back = ops.dequantize8(b, torch.bfloat16)
        assert torch.equal(back[-7:], ops.dequantize8(want, torch.bfloat16))
        assert not back[:-7].any()
        del b, back
        torch.cuda.empty_cache()
