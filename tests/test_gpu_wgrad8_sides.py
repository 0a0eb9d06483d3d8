"""The weight gradient's kernels of 128- and 256-wide tiles, in one slice of the batch and in several;
which one runs is asserted.

Bounds: every product is exact; a sum takes one addition for each of the batch's rows and each part of
dz (three of float32, two of float16), 64 more for the slices, each 2^-24 of the sum of magnitudes."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.routes8 import wgrad8_plan
from tests.test_gpu_block8 import U, _dtype, _normal, _values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


# ragged in the batch, outputs and inputs; the groups of four tiles end whole and ragged
SIZES = {(1030, 770, 900): (128, 4), (6000, 250, 790): (128, 19), (200, 2050, 2050): (128, 1),
         (33, 3801, 3700): (128, 1), (4100, 2050, 1800): (256, 3), (100, 4100, 4000): (256, 1),
         (8200, 1100, 2000): (256, 6)}


def _bounds(dz, x, dtype):
    import torch
    z, v = dz.double(), torch.from_numpy(_values(x)).cuda()
    n = dz.shape[0] * {"f32": 3, "f16": 2, "bf16": 1}[dtype] + 64
    zt = z.t().contiguous()
    return zt @ v, n * U * (zt.abs() @ v.abs()) + 2.0 ** -140, z.sum(0), n * U * z.abs().sum(0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", list(SIZES))
def test_weight_gradient(size, dtype):
    import torch
    from cudeep_amd import ops
    M, N, K = size
    assert wgrad8_plan(M, N, K) == SIZES[size]
    dz = (_normal((M, N), 51) * M ** -0.5).to(_dtype(dtype))
    x = ops.quantize8(_normal((M, K), 52))
    say("linear_weight_grad8", size, dtype)
    dw, db = ops.linear_weight_grad8(dz, x)
    want, bound, want_b, bound_b = _bounds(dz, x, dtype)
    assert ((dw.double() - want).abs() <= bound).all()
    assert ((db.double() - want_b).abs() <= bound_b).all()
    # alone, and again: the same bits
    dw2, none = ops.linear_weight_grad8(dz, x, bias=False)
    assert none is None and torch.equal(dw2, dw)
    again = ops.linear_weight_grad8(dz, x)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", list(SIZES))
def test_whole_numbers(size, dtype):
    """Every sum is exact in fp32, whatever its order."""
    import torch
    from cudeep_amd import ops
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(6)
    dz = torch.randint(-8, 9, (M, N), device="cuda", generator=g).to(_dtype(dtype))
    xv = torch.randint(-8, 9, (M, K), device="cuda", generator=g).float()
    say("linear_weight_grad8 whole numbers", size, dtype)
    dw, db = ops.linear_weight_grad8(dz, ops.quantize8(xv))
    assert torch.equal(dw.double(), dz.double().t().contiguous() @ xv.double())
    assert torch.equal(db.double(), dz.double().sum(0))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [(1030, 770, 900), (4100, 2050, 1800)])
def test_faults_and_strides(size, dtype):
    """Infinities and NaN reach their own row or column of the gradient alone; the same bits from
    views that begin at odd elements and bytes, with NaN around."""
    import torch
    from cudeep_amd import ops
    M, N, K = size
    wide = torch.full((M, N + 21), float("nan"), device="cuda", dtype=_dtype(dtype))
    dz = wide[:, 3:3 + N]
    dz.copy_(_normal((M, N), 71))
    x = ops.quantize8(_normal((M, K), 72))
    q = torch.full((M, K + 5), 0x7f, dtype=torch.uint8, device="cuda")
    q[:, 1:K + 1] = x.q.view(torch.uint8)
    s = torch.full((M, x.scale.shape[1] + 1), 255, dtype=torch.uint8, device="cuda")
    s[:, 1:] = x.scale.view(torch.uint8)
    x2 = ops.Block8(q.view(torch.float8_e4m3fn)[:, 1:K + 1], s.view(torch.float8_e8m0fnu)[:, 1:], 1)
    say("linear_weight_grad8 faults and strides", size, dtype)
    clean = ops.linear_weight_grad8(dz.contiguous(), x)
    for a, b in zip(ops.linear_weight_grad8(dz, x2), clean):
        assert torch.equal(a, b)
    dz[M - 1, 5], dz[3, N - 1] = float("inf"), float("nan")
    q[7, 1 + K - 2] = 0x7f
    s[9, 1] = 255    # a scale: 128 columns
    dw, db = ops.linear_weight_grad8(dz, x2)
    assert not dw[5].isfinite().any() and dw[N - 1].isnan().all() and db[5].isinf() and db[N - 1].isnan()
    assert dw[:, K - 2].isnan().all() and dw[:, :128].isnan().all()
    for t in (dw, clean[0]):
        t[5] = t[N - 1] = 0
        t[:, K - 2] = 0
        t[:, :128] = 0
    for t in (db, clean[1]):
        t[5] = t[N - 1] = 0
    assert torch.equal(dw, clean[0]) and torch.equal(db, clean[1])


@pytest.mark.parametrize("size", [(1030, 770, 900), (4100, 2050, 1800)])
def test_wide_ranges(size):
    """fp32 gradients of 24 bits over many powers of two in one row of the batch, the other rows zero:
    the product's rounding is all there is, and the largest finite values stay finite."""
    import torch
    from cudeep_amd import ops
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(16)
    dz = torch.zeros((M, N), device="cuda")
    dz[M - 3] = torch.randn(N, device="cuda", generator=g) * torch.exp2(
        torch.randint(-60, 60, (N,), device="cuda", generator=g).float())
    dz[M - 3, 0], dz[M - 3, 9] = torch.finfo(torch.float32).max, -3.39e38
    x = ops.quantize8(torch.full((M, K), 0.5, device="cuda"))
    say("linear_weight_grad8 wide ranges", size)
    dw, db = ops.linear_weight_grad8(dz, x)
    assert torch.equal(dw, (dz[M - 3] * 0.5)[:, None].expand(N, K)) and torch.equal(db, dz[M - 3])


def test_offsets_beyond_32_bits():
    """A batch whose gradients take more than 2^32 bytes: its last rows alone are not zero."""
    import torch
    from cudeep_amd import ops
    M, N, K = 1 << 20, 2100, 130
    assert wgrad8_plan(M, N, K)[0] == 256
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("needs 20 GB of device memory")
    dz = torch.zeros((M, N), device="cuda", dtype=torch.bfloat16)
    tail, xt = _normal((50, N), 1).to(torch.bfloat16), _normal((50, K), 2)
    dz[-50:] = tail
    xv = torch.ones((M, K), device="cuda")
    xv[-50:] = xt
    say("linear_weight_grad8", M, N, K)
    dw, db = ops.linear_weight_grad8(dz, ops.quantize8(xv))
    want, bound, want_b, bound_b = _bounds(tail, ops.quantize8(xt), "bf16")
    assert ((dw.double() - want).abs() <= bound).all()
    assert ((db.double() - want_b).abs() <= bound_b).all()
