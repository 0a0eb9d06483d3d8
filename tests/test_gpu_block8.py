"""The 8-bit block-scaled format on the GPU: quantiser, products, activations and weight gradients
against tests/block8_ref.py and 64-bit sums.

Codes, scales and restored values are compared exactly.  Products: a code times a code is exact in
fp32 and so is a part of dz times a restored input, so that only the additions round, at most
2^-24 of the sum of magnitudes for each of a chain's additions; the chain is at most the sum's
length.  A float scale adds two roundings to each block's sum; the output's type half a unit in
its last place.  Products with results of 16 bits run on the 8-bit matrix instruction, which adds
eight products (consecutive k) on a grid 2^-13 below the power of two of the largest: each loses less
than 2^-13 of the largest, eight of them less than 2^-10."""
import numpy as np
import pytest

from tests import block8_ref as ref
from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _ops():
    import cudeep_amd.ops as o
    return o


def _dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
            "e8m0": torch.float8_e8m0fnu}[name]


def _half_ulp(dtype):
    import torch
    return {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]


def _codes(b):
    import torch
    return b.q.view(torch.uint8).cpu().numpy()


def _scales(b):
    """A Block8's scales as float64."""
    import torch
    if b.scale.dtype == torch.float32:
        return b.scale.cpu().numpy().astype(np.float64)
    return 2.0 ** (b.scale.view(torch.uint8).cpu().numpy().astype(np.float64) - 127)


def _values(b):
    return ref.values(_codes(b), _scales(b), b.tile_rows)


def _normal(shape, seed, spread=0.5):
    """Values whose columns differ in size, on the device in float32."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g) * \
        torch.exp(spread * torch.randn((1, shape[1]), device="cuda", generator=g))


# ---- quantiser -------------------------------------------------------------------------------

SIZES = [(1, 1), (1, 4096), (3, 7), (5, 127), (130, 128), (9, 129), (257, 255), (37, 1000),
         (64, 333), (129, 640)]


@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", SIZES)
def test_quantize(size, dtype, scale):
    import torch
    ops = _ops()
    x = (_normal(size, sum(size)) * 3).to(_dtype(dtype))
    for tile_rows in (1, 128):
        say("quantize", size, dtype, scale, tile_rows)
        b = ops.quantize8(x, tile_rows, scale_dtype=_dtype(scale))
        codes, exps = ref.quantize(x.double().cpu().numpy(), tile_rows)
        assert np.array_equal(_codes(b), codes)
        assert np.array_equal(_scales(b), 2.0 ** exps)
        for out in ("f32", "bf16", "f16"):
            back = ops.dequantize8(b, _dtype(out))
            want = torch.from_numpy(ref.values(codes, 2.0 ** exps, tile_rows)).to(_dtype(out))
            assert torch.equal(back.cpu(), want)


def test_quantize_special_values():
    """Zeros, powers of two at the scale's edges, ties, subnormals, the largest and the smallest
    numbers, infinities and NaN, each in a block of its own."""
    import torch
    ops = _ops()
    f = np.float32
    blocks = [
        [0.0, -0.0], [448.0, 1.0], [np.nextafter(f(448), f(500)), 1.0], [449.0 * 2 ** -9, 3.0],
        [447.9, 17.0, 18.0, 19.0, 20.0, -17.0, -19.0, 0.0146484375, 2 ** -9, 2 ** -10, 3 * 2 ** -11, -2 ** -10],
        [f(3.4028235e38), 1e38, 1.0], [f(2 ** -149), 0.0], [f(1e-40), f(1e-38)],
        [448 * 2.0 ** -117, 2.0 ** -117], [448 * 2.0 ** -118, 2.0 ** -126],
        [np.inf, 1.0, 448.0], [-np.inf, np.nan, 0.5], [np.nan], [np.inf], [np.nan, 0.0],
    ]
    x = np.zeros((len(blocks), 128), np.float32)
    for i, v in enumerate(blocks):
        x[i, :len(v)] = v
    say("quantize special values")
    for tile_rows in (1, 128):
        b = ops.quantize8(torch.from_numpy(x).cuda(), tile_rows)
        codes, exps = ref.quantize(x, tile_rows)
        got = _codes(b)
        nan = codes & 127 == 127
        assert np.array_equal(got & 127 == 127, nan)
        assert np.array_equal(got[~nan], codes[~nan])
        assert np.array_equal(_scales(b), 2.0 ** exps)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_quantize_strided(dtype):
    """Views that begin at odd elements, as inputs and as operands."""
    import torch
    ops = _ops()
    wide = (_normal((65, 700), 4)).to(_dtype(dtype))
    view = wide[:, 5:5 + 333]
    a, b = ops.quantize8(view), ops.quantize8(view.contiguous())
    assert np.array_equal(_codes(a), _codes(b)) and np.array_equal(_scales(a), _scales(b))
    out = torch.full((65, 400), 9.0, device="cuda")
    ops.dequantize8(a, out=out[:, 1:334])
    assert torch.equal(out[:, 1:334], ops.dequantize8(b))
    assert (out[:, 0] == 9).all() and (out[:, 334:] == 9).all()
    assert ops.quantize8(wide[:0]).q.shape == (0, 700)


# ---- products ----------------------------------------------------------------------------------

def _operands(M, N, K, scale, seed):
    """Block8 operands; float scales are no powers of two."""
    import torch
    ops = _ops()
    a = ops.quantize8(_normal((M, K), seed), scale_dtype=_dtype(scale))
    b = ops.quantize8(_normal((N, K), seed + 1) * K ** -0.5, 128, scale_dtype=_dtype(scale))
    if scale == "f32":
        g = torch.Generator(device="cuda").manual_seed(seed + 2)
        for s in (a.scale, b.scale):
            s.mul_(1 + torch.rand(s.shape, device="cuda", generator=g))
    return a, b


def _grid_loss(a, b):
    """The 8-bit instruction's loss: 2^-10 of the largest of each eight products, on the device."""
    import torch
    M, K = a.shape
    pad = ((0, 0), (0, -K % 8))
    a, b = (torch.from_numpy(np.pad(np.abs(t), pad)).float().cuda().view(t.shape[0], -1, 8) for t in (a, b))
    loss = torch.zeros((M, b.shape[0]), device="cuda")
    for k in range(a.shape[1]):
        loss += (a[:, None, k] * b[None, :, k]).amax(-1)
    return loss.double().cpu().numpy() * 2.0 ** -10


def _check_product(got, a, b, bias, act, K):
    """got against act(A B^T + bias) of float64 matrices."""
    import torch
    exact = a @ b.T
    mag = np.abs(a) @ np.abs(b).T
    if bias is not None:
        exact = exact + bias
        mag = mag + np.abs(bias)
    bound = (K + 8) * U * mag
    if got.dtype != torch.float32 and K:
        bound = bound + _grid_loss(a, b)
    if act == "relu":
        exact = np.maximum(exact, 0)
    elif act in ("gelu", "silu", "sigmoid"):
        # slopes of at most 1.13, and a few roundings of the function itself (the exponent's
        # argument is rounded: 2^-24 of its size, which the function's tails make harmless)
        bound = 1.13 * bound + 16 * U * (np.abs(exact) + 1)
        u = 0.7978845608 * (exact + 0.044715 * exact ** 3) * 2 if act == "gelu" else exact
        with np.errstate(over="ignore"):
            exact = (1 if act == "sigmoid" else exact) / (1 + np.exp(-u))
    bound = bound + _half_ulp(got.dtype) * np.abs(exact) + 2.0 ** -25
    over = (np.abs(got.double().cpu().numpy() - exact) - bound).max() if exact.size else -1
    assert over <= 0, over


# token counts at and around the tiles' edges; inner sizes of no whole block, of less than a
# 16-byte piece, and long ones with few outputs
PRODUCTS = [(1, 1, 1), (1, 16, 128), (1, 300, 1000), (1, 4096, 512), (2, 129, 127), (5, 64, 129),
            (7, 130, 4096), (16, 512, 384), (17, 257, 640), (31, 96, 4099), (33, 1000, 1200),
            (64, 64, 256), (65, 63, 333), (100, 320, 96), (128, 128, 128), (129, 130, 131),
            (200, 48, 2048), (255, 257, 512), (256, 256, 1024), (300, 640, 777), (515, 512, 256),
            (1025, 384, 144), (640, 1300, 400)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("size", PRODUCTS)
def test_product(size, scale, dtype):
    import torch
    ops = _ops()
    M, N, K = size
    a, b = _operands(M, N, K, scale, M + N + K)
    say("gemm8", size, scale, dtype)
    got = ops.gemm8(a, b, dtype=_dtype(dtype))
    _check_product(got, _values(a), _values(b), None, "none", K)
    assert torch.equal(got, ops.gemm8(a, b, dtype=_dtype(dtype)))


@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("size", PRODUCTS + [(2048, 1280, 520), (770, 2050, 1152)])
def test_product_of_whole_numbers(size, scale):
    """Small whole numbers under scales of a few powers of two: every sum is exact in fp32, whatever
    its order, on either matrix instruction, and is rounded once to the result's type."""
    import torch
    ops = _ops()
    M, N, K = size
    g = torch.Generator(device="cuda").manual_seed(K)

    def whole(rows, tiles, most, tile_rows):
        q = torch.randint(-most, most + 1, (rows, K), device="cuda", generator=g).float()
        e = torch.randint(-2, 3, (tiles, -(-K // 128)), device="cuda", generator=g)
        s = (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
        return ops.Block8(q.to(torch.float8_e4m3fn), s if scale == "e8m0" else torch.exp2(e.float()),
                          tile_rows)

    a, b = whole(M, M, 2, 1), whole(N, -(-N // 128), 3, 128)
    exact = torch.from_numpy(_values(a) @ _values(b).T)
    say("gemm8 whole numbers", size, scale)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        assert torch.equal(ops.gemm8(a, b, dtype=dt).cpu(), exact.to(torch.float32).to(dt)), dt


# more tiles, and blocks in a ring of buffers: fewer blocks than buffers, a panel of scales that ends
# before the last block, ragged tiles and a ragged last block
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("size", [(1000, 1100, 128), (300, 4096, 256), (520, 2000, 384), (40, 70, 2048),
                                  (129, 130, 2176), (33, 65, 4224), (70, 200, 8320), (1100, 2300, 512),
                                  (1025, 2176, 2500), (3590, 3601, 300), (3601, 3590, 2432)])
def test_product_by_many_tiles(size, scale, dtype):
    import torch
    ops = _ops()
    M, N, K = size
    a, b = _operands(M, N, K, scale, 7)
    say("gemm8 tiles", size, scale, dtype)
    got = ops.gemm8(a, b, dtype=_dtype(dtype))
    _check_product(got, _values(a), _values(b), None, "none", K)
    # operands and result inside larger ones
    q = torch.zeros((M, K + 16), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    q[:, :K] = a.q
    out = torch.zeros((M, N + 3), device="cuda", dtype=_dtype(dtype))
    ops.gemm8(ops.Block8(q[:, :K], a.scale), b, dtype=_dtype(dtype), out=out[:, 1:N + 1])
    assert torch.equal(out[:, 1:N + 1], got) and not out[:, 0].any() and not out[:, N + 1:].any()


# the ring's last block without whole pieces, after whole panels of scales and inside one
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("size", [(64, 100, 2064), (40, 70, 4200), (100, 130, 8200), (512, 2050, 144)])
def test_product_by_ragged_blocks(size, scale, dtype):
    import torch
    ops = _ops()
    M, N, K = size
    a, b = _operands(M, N, K, scale, 7)
    say("gemm8 ragged blocks", size, scale, dtype)
    got = ops.gemm8(a, b, dtype=_dtype(dtype))
    _check_product(got, _values(a), _values(b), None, "none", K)
    # what lies behind the last column is not read as codes (0x7f is NaN)
    wide = torch.full((M, a.q.stride(0) + 16), 0x7f, device="cuda", dtype=torch.uint8)
    wide = wide.view(torch.float8_e4m3fn)
    wide[:, :K] = a.q
    assert torch.equal(ops.gemm8(ops.Block8(wide[:, :K], a.scale), b, dtype=_dtype(dtype)), got)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("size", [(1, 333, 640), (40, 130, 2048), (300, 260, 250), (600, 2048, 300)])
def test_epilogues_of_16_bits(size, act, dtype):
    ops = _ops()
    from cudeep_amd import _lib as L
    M, N, K = size
    epi = {"relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU, "sigmoid": L.EPI_SIGMOID}[act]
    a, b = _operands(M, N, K, "e8m0", 3)
    bias = _normal((1, N), 9)[0]
    say("gemm8 epilogue", size, act, dtype)
    got = ops.gemm8(a, b, bias=bias, epilogue=epi, dtype=_dtype(dtype))
    _check_product(got, _values(a), _values(b), bias.double().cpu().numpy(), act, K)


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu", "sigmoid"])
@pytest.mark.parametrize("size", [(1, 333, 640), (40, 130, 1000), (300, 260, 256), (600, 1024, 300)])
def test_epilogues(size, act):
    import torch
    ops = _ops()
    from cudeep_amd import _lib as L
    M, N, K = size
    epi = {"none": L.EPI_NONE, "relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU,
           "sigmoid": L.EPI_SIGMOID}[act]
    a, b = _operands(M, N, K, "e8m0", 3)
    bias = _normal((1, N), 9)[0]
    say("gemm8 epilogue", size, act)
    got = ops.gemm8(a, b, bias=bias, epilogue=epi, dtype=torch.float32)
    _check_product(got, _values(a), _values(b), bias.double().cpu().numpy(), act, K)
    # the same from the unquantised input, and the sum over no columns
    x = ops.dequantize8(a)
    assert torch.equal(ops.linear8(x, b, bias, epilogue=epi), got)
    none = ops.gemm8(ops.Block8(a.q[:, :0], a.scale[:, :0]), ops.Block8(b.q[:, :0], b.scale[:, :0], 128),
                     bias=bias, epilogue=epi, dtype=torch.float32)
    _check_product(none, np.zeros((M, 0)), np.zeros((N, 0)), bias.double().cpu().numpy(), act, 0)


@pytest.mark.parametrize("size", [(1, 200, 1000), (3, 4096, 1024), (16, 130, 777), (64, 256, 512),
                                  (130, 300, 640), (520, 512, 1030)])
@pytest.mark.parametrize("scale", ["e8m0", "f32"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_linear(size, scale, dtype):
    """linear8(x) is gemm8(quantize8(x)) bit for bit."""
    import torch
    ops = _ops()
    M, N, K = size
    x = _normal((M, K), 5).to(_dtype(dtype))
    b = _operands(1, N, K, scale, 6)[1]
    bias = _normal((1, N), 7)[0]
    say("linear8", size, scale, dtype)
    got = ops.linear8(x, b, bias)
    assert got.dtype == x.dtype
    a = ops.quantize8(x, scale_dtype=_dtype(scale))
    assert torch.equal(got, ops.gemm8(a, b, bias=bias, dtype=x.dtype))
    _check_product(got, _values(a), _values(b), bias.double().cpu().numpy(), "none", K)


@pytest.mark.parametrize("size", [(1, 300, 500), (50, 260, 700), (300, 300, 600), (512, 512, 640)])
@pytest.mark.parametrize("shift", [1, 4, 16])
def test_unaligned_operands(size, shift):
    """Codes whose rows begin at any byte, scales and outputs inside wider matrices."""
    import torch
    ops = _ops()
    M, N, K = size
    a, b = _operands(M, N, K, "e8m0", 8)
    want = ops.gemm8(a, b, dtype=torch.bfloat16)

    def inside(t, pad):
        wide = torch.zeros((t.shape[0], t.shape[1] + pad + shift), dtype=torch.uint8, device="cuda")
        wide.fill_(0x7f)   # NaN codes around: nothing beside the view may be used
        wide[:, shift:shift + t.shape[1]] = t.view(torch.uint8)
        return wide.view(t.dtype)[:, shift:shift + t.shape[1]]

    a2 = ops.Block8(inside(a.q, 3), inside(a.scale, 1), 1)
    b2 = ops.Block8(inside(b.q, 5), inside(b.scale, 2), 128)
    out = torch.full((M, N + 7), 5.0, device="cuda", dtype=torch.bfloat16)
    say("gemm8 unaligned", size, shift)
    got = ops.gemm8(a2, b2, out=out[:, 3:3 + N])
    assert torch.equal(got, want)
    assert (out[:, :3] == 5).all() and (out[:, 3 + N:] == 5).all()


def test_faults_stay_in_their_rows_and_columns():
    import torch
    ops = _ops()
    for M, N, K in ((4, 200, 384), (150, 200, 384), (600, 512, 512)):
        x = _normal((M, K), 1)
        w = _normal((N, K), 2)
        clean = ops.linear8(x, ops.quantize8(w, 128))
        x[1, 200] = float("inf")
        w[7, 3] = float("nan")
        say("linear8 faults", M, N, K)
        got = ops.linear8(x, ops.quantize8(w, 128))
        assert got[1].isnan().all() and got[:, 7].isnan().all()
        keep = torch.ones((M, N), dtype=torch.bool, device="cuda")
        keep[1] = False
        keep[:, 7] = False
        # (the weights' scale looks at the others alone, so it is as it was if column 3 of row 7 was
        # not its tile's largest)
        assert got[keep].isfinite().all() and torch.equal(got[keep], clean[keep])


def test_extreme_scales():
    """The scale bytes' ends: products of the largest and the smallest scales, zero-scale float
    blocks, and a NaN scale, which makes its row (its tile's columns) NaN."""
    import torch
    ops = _ops()
    M, N, K = 40, 130, 256
    a, b = _operands(M, N, K, "e8m0", 12)
    sa, sb = a.scale.view(torch.uint8), b.scale.view(torch.uint8)
    sa[:, 0], sb[:, 0] = 240, 20     # 2^113 * 2^-107
    sa[:, 1], sb[:, 1] = 14, 246     # 2^-113 * 2^119
    say("gemm8 extreme scales")
    _check_product(ops.gemm8(a, b, dtype=torch.float32), _values(a), _values(b), None, "none", K)
    sa[5, 1] = 255
    got = ops.gemm8(a, b, dtype=torch.float32)
    assert got[5].isnan().all() and got[:5].isfinite().all() and got[6:].isfinite().all()
    a, b = _operands(M, N, K, "f32", 12)
    a.scale[3, 0] = 0.0
    b.scale[1, 1] = float("nan")
    got = ops.gemm8(a, b, dtype=torch.float32)
    assert got[:, 128:].isnan().all()
    va = _values(a)
    _check_product(got[:, :128], va, _values(b)[:128], None, "none", K)


def test_product_offsets_beyond_32_bits():
    """Rows of a weight and of an output more than 2^32 bytes in."""
    import torch
    ops = _ops()
    free, _ = torch.cuda.mem_get_info()
    if free < 30 << 30:
        pytest.skip("needs 30 GB of device memory")
    K, N = 4096, (1 << 20) + 77
    w = ops.Block8(torch.zeros((N, K), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
                   torch.full((-(-N // 128), K // 128), 127, dtype=torch.uint8,
                              device="cuda").view(torch.float8_e8m0fnu), 128)
    tail = ops.quantize8(_normal((77, K), 3), 128)
    w.q.view(torch.uint8)[-77:] = tail.q.view(torch.uint8)
    w.scale.view(torch.uint8)[-1:] = tail.scale.view(torch.uint8)
    for M in (2, 1200):
        x = ops.quantize8(_normal((M, K), 4))
        say("gemm8 large", M, N, K)
        got = ops.gemm8(x, w, dtype=torch.float32)
        want = ops.gemm8(x, tail, dtype=torch.float32)
        torch.cuda.synchronize()
        # (another kernel may take the small product: its sums in another order)
        mag = np.abs(_values(x)) @ np.abs(_values(tail)).T
        assert (np.abs((got[:, -77:] - want).double().cpu().numpy()) <= 2 * K * U * mag).all()
        assert not got[:, :1000].any()
        del got


# ---- activations ---------------------------------------------------------------------------------

ACTS = ["relu", "gelu", "silu", "sigmoid", "tanh", "leaky"]


def _act64(v, act):
    with np.errstate(over="ignore"):
        if act == "relu":
            return np.where(v > 0, v, 0.0), (v > 0).astype(float)
        if act == "leaky":
            return np.where(v > 0, v, 0.25 * v), np.where(v > 0, 1.0, 0.25)
        if act == "tanh":
            t = np.tanh(v)
            return t, (1 - t) * (1 + t)
        z = v if act != "gelu" else 2 * 0.7978845608 * (v + 0.044715 * v ** 3)
        s, r = 1 / (1 + np.exp(-z)), 1 / (1 + np.exp(z))
        if act == "sigmoid":
            return s, s * r
        dz = 1 if act == "silu" else 2 * 0.7978845608 * (1 + 3 * 0.044715 * v ** 2)
        return v * s, s + v * s * r * dz


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("size", [(1, 1), (3, 130), (70, 1000), (33, 512)])
def test_activation(size, act, dtype):
    import torch
    ops = _ops()
    from cudeep_amd import _lib as L
    code = {"relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU, "sigmoid": L.EPI_SIGMOID,
            "tanh": L.ACT_TANH, "leaky": L.ACT_LEAKY_RELU}[act]
    dt = _dtype(dtype)
    z = (2 * _normal(size, 31)).to(dt)
    dy = _normal(size, 32).to(dt)
    say("activation8", size, act, dtype)
    y, kept = ops.activation8(z, code, alpha=0.25)
    codes, exps = ref.quantize(z.double().cpu().numpy())
    assert np.array_equal(_codes(kept), codes) and np.array_equal(_scales(kept), 2.0 ** exps)
    dz = ops.activation_backward8(dy, kept, code, alpha=0.25)
    # functions: a handful of roundings, the exponent's argument 2^-24 of its size (the hardware
    # functions add 2^-22), relative to values of at most |v| and slopes of at most 1.13
    f = (64 if dtype != "f32" else 16) * U
    for got, at, fac, pick in ((y, z.double().cpu().numpy(), 1.0, 0),
                               (dz, _values(kept), dy.double().cpu().numpy(), 1)):
        v = _act64(at, act)[pick]
        exact = v * fac
        bound = (f * (1 + np.abs(at)) * np.abs(fac) if act not in ("relu", "leaky") else U * np.abs(exact))
        bound = bound + _half_ulp(dt) * np.abs(exact) + 2.0 ** -25
        over = (np.abs(got.double().cpu().numpy() - exact) - bound).max()
        assert over <= 0, over


def test_activation_tails():
    """Large arguments: no NaN where the exponentials overflow; infinities and NaN are kept."""
    import torch
    ops = _ops()
    from cudeep_amd import _lib as L
    v = torch.tensor([[-3e4, -200.0, -89.0, -20.0, 0.0, 20.0, 89.0, 200.0, 3e4]], device="cuda")
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        z = v.to(dt, copy=True)
        one = torch.ones_like(z)
        for code in (L.EPI_RELU, L.EPI_GELU, L.EPI_SILU, L.EPI_SIGMOID, L.ACT_TANH):
            y, kept = ops.activation8(z, code)
            dz = ops.activation_backward8(one, kept, code)
            assert y.isfinite().all() and dz.isfinite().all()
            if code in (L.EPI_RELU, L.EPI_GELU, L.EPI_SILU):
                # (SiLU's slope at -89 is -89 e^-89, about 1e-37)
                assert (y[0, :3].float().abs() < 1e-30).all() and torch.equal(y[0, 6:], z[0, 6:])
                assert (dz[0, :3].float().abs() < 1e-30).all() and (dz[0, 6:] == 1).all()
        z[0, 4] = float("nan")
        y, kept = ops.activation8(z, L.EPI_GELU)
        assert y[0, 4].isnan() and ops.activation_backward8(one, kept, L.EPI_GELU)[0, 4].isnan()


@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid", "tanh"])
def test_activation_gradient_against_differences(act):
    """(act(v + h) - act(v - h)) / 2h of the framework's own elementwise activation at the restored
    values; h is a power of two that moves them exactly."""
    import torch
    ops = _ops()
    from cudeep_amd import _lib as L
    code = {"gelu": L.EPI_GELU, "silu": L.EPI_SILU, "sigmoid": L.EPI_SIGMOID, "tanh": L.ACT_TANH}[act]
    _, kept = ops.activation8(_normal((20, 256), 41), code)
    v = ops.dequantize8(kept)
    h = 2.0 ** -6
    own = (ops.activation(v + h, code).double() - ops.activation(v - h, code).double()) / (2 * h)
    got = ops.activation_backward8(torch.ones_like(v), kept, code).double()
    at = v.double().cpu().numpy()
    trunc = np.abs((_act64(at + h, act)[0] - _act64(at - h, act)[0]) / (2 * h) - _act64(at, act)[1])
    noise = 32 * U * (1 + np.abs(at)) / h
    assert (np.abs((own - got).cpu().numpy()) <= trunc + noise).all()


# ---- weight gradients -------------------------------------------------------------------------------

GRADS = [(1, 1, 1), (1, 16, 128), (2, 5, 7), (31, 64, 64), (32, 65, 129), (33, 130, 200),
         (64, 250, 333), (100, 10, 256), (257, 128, 128), (300, 256, 784), (1000, 33, 100),
         (2049, 256, 130), (4099, 40, 72), (700, 300, 513), (520, 512, 640)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", GRADS)
def test_weight_gradient(size, dtype):
    import torch
    ops = _ops()
    M, N, K = size
    dz = (_normal((M, N), 51) * M ** -0.5).to(_dtype(dtype))
    x = ops.quantize8(_normal((M, K), 52))
    say("linear_weight_grad8", size, dtype)
    dw, db = ops.linear_weight_grad8(dz, x)
    z, v = dz.double().cpu().numpy(), _values(x)
    # three parts of an fp32 value make three additions to a sum
    n = M * (3 if dtype == "f32" else 2 if dtype == "f16" else 1) + 64
    assert (np.abs(dw.double().cpu().numpy() - z.T @ v) <= n * U * (np.abs(z).T @ np.abs(v)) + 2.0 ** -140).all()
    assert (np.abs(db.double().cpu().numpy() - z.sum(0)) <= n * U * np.abs(z).sum(0)).all()
    # alone, and again: the same bits
    dw2, none = ops.linear_weight_grad8(dz, x, bias=False)
    assert none is None and torch.equal(dw2, dw)
    again = ops.linear_weight_grad8(dz, x)
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


def test_weight_gradient_is_exact_on_whole_numbers():
    """Small whole numbers: every sum is exact in fp32, whatever its order."""
    import torch
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(6)
    for M, N, K in ((77, 100, 200), (600, 520, 520)):
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            dz = torch.randint(-8, 9, (M, N), device="cuda", generator=g).to(dtype)
            xv = torch.randint(-8, 9, (M, K), device="cuda", generator=g).float()
            dw, db = ops.linear_weight_grad8(dz, ops.quantize8(xv))
            assert torch.equal(dw.double().cpu(), dz.double().cpu().T @ xv.double().cpu())
            assert torch.equal(db.double(), dz.double().sum(0))


def test_weight_gradient_of_wide_ranges():
    """fp32 gradients of 24 significant bits over many powers of two: one row at a time, so
    that the product's own rounding is all there is."""
    import torch
    ops = _ops()
    N, K = 200, 130
    g = torch.Generator(device="cuda").manual_seed(16)
    dz = torch.randn((1, N), device="cuda", generator=g) * torch.exp2(
        torch.randint(-60, 60, (1, N), device="cuda", generator=g).float())
    x = ops.quantize8(_normal((1, K), 17))
    dw, db = ops.linear_weight_grad8(dz, x)
    want = dz.double().cpu().numpy().T @ _values(x)
    assert (np.abs(dw.double().cpu().numpy() - want) <= 3 * U * np.abs(want)).all()
    assert torch.equal(db, dz[0])


def test_weight_gradient_faults_and_ends():
    """Infinities and NaN reach their own column alone; the largest finite values stay finite."""
    import torch
    ops = _ops()
    M, N, K = 40, 70, 130
    dz = _normal((M, N), 61)
    xv = _normal((M, K), 62)
    x = ops.quantize8(xv)
    clean, _ = ops.linear_weight_grad8(dz, x)
    dz[3, 5] = float("inf")
    dz[4, 9] = float("nan")
    dw, db = ops.linear_weight_grad8(dz, x)
    assert not dw[5].isfinite().any() and dw[9].isnan().all() and db[5].isinf() and db[9].isnan()
    keep = [n for n in range(N) if n not in (5, 9)]
    assert torch.equal(dw[keep], clean[keep])
    xv[0, 7] = float("nan")
    dw, _ = ops.linear_weight_grad8(_normal((M, N), 61), ops.quantize8(xv))
    assert dw[:, 7].isnan().all() and dw[:, :7].isfinite().all() and dw[:, 8:].isfinite().all()
    one = torch.full((1, 3), torch.finfo(torch.float32).max, device="cuda")
    one[0, 1] = -3.39e38
    dw, db = ops.linear_weight_grad8(one, ops.quantize8(torch.full((1, 9), 0.5, device="cuda")))
    assert torch.equal(dw, (one * 0.5).T.expand(3, 9)) and torch.equal(db, one[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_weight_gradient_strided(dtype):
    import torch
    ops = _ops()
    M, N, K = 150, 77, 201
    wide = _normal((M, N + 20), 71).to(_dtype(dtype))
    dz = wide[:, 3:3 + N]
    x = ops.quantize8(_normal((M, K), 72))
    q = torch.full((M, K + 5), 0x7f, dtype=torch.uint8, device="cuda")
    q[:, 1:K + 1] = x.q.view(torch.uint8)
    x2 = ops.Block8(q.view(torch.float8_e4m3fn)[:, 1:K + 1], x.scale, 1)
    for a, b in zip(ops.linear_weight_grad8(dz, x2), ops.linear_weight_grad8(dz.contiguous(), x)):
        assert torch.equal(a, b)


def test_weight_gradient_along_a_direction():
    """The product is linear in its weight: sum dz (x (W + V)^T - x W^T) is sum V dw, with the
    framework's fp32 product as the forward pass."""
    import torch
    ops = _ops()
    M, N, K = 300, 60, 200
    dz, x = _normal((M, N), 81), ops.quantize8(_normal((M, K), 82))
    xv = ops.dequantize8(x)
    v = _normal((N, K), 83)
    dw, _ = ops.linear_weight_grad8(dz, x)
    y = ops.gemm(xv, v, transB=True).double()
    mag = (dz.abs().double().cpu() * (xv.abs().double().cpu() @ v.abs().double().cpu().T)).sum()
    diff = ((dz.double() * y).sum() - (dw.double() * v.double()).sum()).abs().cpu()
    assert diff <= (M * 3 + K + 64) * U * mag


def test_empty_sizes():
    import torch
    ops = _ops()
    e8 = torch.float8_e8m0fnu
    x = ops.quantize8(torch.zeros((0, 200), device="cuda"))
    dw, db = ops.linear_weight_grad8(torch.zeros((0, 30), device="cuda"), x)
    assert dw.shape == (30, 200) and not dw.any() and not db.any()
    dz = _normal((20, 30), 5)
    dw, db = ops.linear_weight_grad8(dz, ops.quantize8(torch.zeros((20, 0), device="cuda")))
    assert dw.shape == (30, 0) and torch.allclose(db, dz.sum(0), rtol=1e-5, atol=1e-5)
    dw, db = ops.linear_weight_grad8(dz[:, :0], ops.quantize8(dz))
    assert dw.shape == (0, 30) and db.shape == (0,)
    w = ops.quantize8(_normal((50, 200), 6), 128)
    assert ops.gemm8(x, w).shape == (0, 50)
    assert ops.linear8(torch.zeros((0, 200), device="cuda"), w).shape == (0, 50)
    assert x.scale.dtype == e8


def test_workspace_stream_and_capture():
    """Products and weight gradients on the caller's workspace, on another stream, and captured:
    replays between eager work equal the eager results."""
    import torch
    ops = _ops()
    from cudeep_amd import _lib as L
    for M, N, K in ((1, 512, 1024), (20, 130, 2000), (2100, 256, 784)):
        x, dz = _normal((M, K), 91), _normal((M, N), 92)
        w = ops.quantize8(_normal((N, K), 93), 128)
        bias = _normal((1, N), 94)[0]
        ws = torch.empty(max(ops.linear8_workspace_bytes(M, N, K), 1), dtype=torch.uint8, device="cuda")
        wg = torch.empty(max(ops.linear_weight_grad8_workspace_bytes(M, N, K), 1), dtype=torch.uint8,
                         device="cuda")

        def step(x):
            y = ops.linear8(x, w, bias, epilogue=L.EPI_GELU, workspace=ws)
            dw, db = ops.linear_weight_grad8(dz, ops.quantize8(x), workspace=wg)
            return y, dw, db

        say("block8 stream and capture", M, N, K)
        want = step(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step(x)
        side.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        if ops.linear8_workspace_bytes(M, N, K) > 1:
            with pytest.raises(Exception, match="workspace"):
                ops.linear8(x, w, workspace=ws[:-1])
        xin = x.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(xin)
        for k in range(4):
            x2 = x * (1 + k)
            xin.copy_(x2)
            graph.replay()
            torch.cuda.synchronize()
            kept = [t.clone() for t in out]
            for a, b in zip(kept, step(x2)):
                assert torch.equal(a, b), k


def test_refusals():
    import torch
    ops = _ops()
    from cudeep_amd import _lib as L
    x = _normal((40, 200), 1)
    a, b = _operands(40, 150, 200, "e8m0", 2)
    q = torch.float8_e4m3fn
    bad = [lambda: ops.quantize8(x.cpu()), lambda: ops.quantize8(x.double()), lambda: ops.quantize8(x.t()),
           lambda: ops.quantize8(x[0]), lambda: ops.quantize8(x, 64),
           lambda: ops.quantize8(x, scale_dtype=torch.float16), lambda: ops.dequantize8(a.q),
           lambda: ops.dequantize8(a, torch.float64), lambda: ops.gemm8(a, a), lambda: ops.gemm8(b, b),
           lambda: ops.gemm8(a, ops.Block8(b.q[:, :199], b.scale, 128)),
           lambda: ops.gemm8(a, b, dtype=torch.float64), lambda: ops.gemm8(a, b, bias=x[0][:149]),
           lambda: ops.gemm8(a, b, bias=x[0][:150].half()), lambda: ops.gemm8(a, b, epilogue=L.ACT_TANH),
           lambda: ops.gemm8(a, b, out=x), lambda: ops.gemm8(ops.Block8(a.q, a.scale[:, :1]), b),
           lambda: ops.gemm8(ops.Block8(a.q.view(torch.uint8), a.scale), b),
           lambda: ops.gemm8(ops.Block8(a.q, a.scale.view(torch.uint8)), b),
           lambda: ops.gemm8(ops.Block8(a.q, a.scale.cpu()), b), lambda: ops.linear8(x[:, :199], b),
           lambda: ops.linear8(x.double(), b), lambda: ops.linear8(x, a),
           lambda: ops.linear8(x.view(2, 20, 200), b), lambda: ops.activation8(x, L.EPI_NONE),
           lambda: ops.activation8(x, 77), lambda: ops.activation8(x[0], L.EPI_RELU),
           lambda: ops.activation_backward8(x[:, :199], a, L.EPI_RELU),
           lambda: ops.activation_backward8(x, a, L.EPI_NONE),
           lambda: ops.linear_weight_grad8(x[:39], a), lambda: ops.linear_weight_grad8(x, b),
           lambda: ops.linear_weight_grad8(x, ops.quantize8(x, scale_dtype=torch.float32)),
           lambda: ops.linear_weight_grad8(x.double(), a)]
    assert a.q.dtype == q
    for k, f in enumerate(bad):
        with pytest.raises((TypeError, ValueError, RuntimeError, AttributeError)):
            f()
            pytest.fail(f"refusal {k} was accepted")
