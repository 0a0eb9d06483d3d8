"""The Linear layer in 16 bits (linear16, linear16_backward) against the formulas in 64 bits.

Bounds.  A product of two 16-bit values is exact in fp32 (22 bits at most); a sum of K of them rounds at
most K times, and slices and the bias a few times more: (K + 8) 2^-24 of the sum of magnitudes.  An
activation has a slope of at most 1.13 and, from the hardware's exponential and reciprocal, a relative
error below 2^-20 of |z| + 1.  A result in 16 bits is off by half a step of its own, eps / 2 of its value
(f16: at least 2^-25, half of the least step).  Backward, dz = grad epi'(z) is such a result, so
that its error goes into the products: |error of dz| times the other operand's magnitudes."""
import numpy as np
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _t():
    import torch
    return torch


def _ops():
    import cudeep_amd.ops as o
    return o


def _dtype(name):
    torch = _t()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _act_code(name):
    from cudeep_amd import _lib as L
    return {"none": L.EPI_NONE, "relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU,
            "sigmoid": L.EPI_SIGMOID}[name]


def _rnd(shape, seed, dtype, scale=1.0):
    torch = _t()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(_dtype(dtype))


def _act(z, act):
    torch = _t()
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * torch.sigmoid(2 * 0.7978845608 * (z + 0.044715 * z ** 3))
    if act == "silu":
        return z * torch.sigmoid(z)
    return torch.sigmoid(z) if act == "sigmoid" else z


def _slope(z, act):
    torch = _t()
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        p = torch.sigmoid(2 * 0.7978845608 * (z + 0.044715 * z ** 3))
        return p + 2 * z * p * (1 - p) * 0.7978845608 * (1 + 3 * 0.044715 * z ** 2)
    p = torch.sigmoid(z)
    if act == "silu":
        return p * (1 + z * (1 - p))
    return p * (1 - p) if act == "sigmoid" else torch.ones_like(z)


def _half(dtype):
    """(half a step relative to a value, half of the least step)"""
    torch = _t()
    return torch.finfo(dtype).eps / 2, 2.0 ** -25 if dtype == torch.float16 else 0.0


def _within(got, want, bound, what):
    if got.numel() == 0:
        return
    rel, least = _half(got.dtype)
    over = ((got.double() - want).abs() - bound - rel * want.abs() - rel * bound - least).max()
    assert float(over) <= 0, (what, float(over))


def _check_forward(x, w, b, act, res, y, z=None):
    K = x.shape[1]
    zx = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if b is not None:
        zx, mag = zx + b.double(), mag + b.double().abs()
    bound = (K + 8) * U * mag
    if z is not None:
        _within(z, zx, bound, "z")
    if act != "none":
        bound = 1.13 * bound + 2.0 ** -20 * (zx.abs() + 1)
    yx = _act(zx, act)
    if res is not None:
        yx = yx + res.double()
    _within(y, yx, bound + 2 * U * yx.abs(), "y")


def _check_backward(dy, x, w, z, act, dx, dw, db):
    M, N = dy.shape
    g = dy.double()
    dz = g if act == "none" else g * _slope(z.double(), act)
    e = g * 0
    if act != "none":
        rel, least = _half(dy.dtype)
        e = (1 + rel) * 2.0 ** -20 * g.abs() * (1 + z.double().abs()) + rel * dz.abs() + least
    a = dz.abs() + e
    if dx is not None:
        wa = w.double().abs()
        _within(dx, dz @ w.double(), e @ wa + (N + 8) * U * (a @ wa), "dx")
    if dw is not None:
        xa = x.double().abs()
        _within(dw, dz.t().contiguous() @ x.double(),
                e.t().contiguous() @ xa + (M + 8) * U * (a.t().contiguous() @ xa), "dw")
    if db is not None:
        _within(db, dz.sum(0), e.sum(0) + (M + 8) * U * a.sum(0), "db")


# rows at and around the tiles' edges, a single one, columns and inner sizes of no whole 8, 16 or 64, a long
# inner size with few outputs, and enough tiles for each kernel
SIZES = [(1, 1, 1), (1, 16, 64), (1, 300, 1000), (1, 1024, 2048), (2, 129, 127), (3, 8, 4104), (5, 64, 130),
         (7, 130, 4096), (16, 512, 384), (17, 257, 640), (31, 96, 4099), (33, 1000, 1200), (48, 2000, 520),
         (64, 64, 256), (65, 63, 333), (100, 320, 96), (127, 264, 72), (128, 128, 128), (129, 136, 136),
         (200, 48, 2048), (255, 257, 512), (256, 256, 1024), (300, 640, 777), (515, 512, 256),
         (1025, 384, 144), (640, 1300, 400), (2048, 264, 200), (1100, 2056, 328)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("size", SIZES)
def test_forward(size, dtype):
    M, N, K = size
    for n, act in enumerate(("none", "relu", "gelu", "silu", "sigmoid")):
        say("linear16", size, dtype, act)
        x, w = _rnd((M, K), 1, dtype), _rnd((N, K), 2, dtype, K ** -0.5)
        b = None if n == 1 else _rnd((N,), 3, "f32" if n == 2 else dtype)
        res = None if n == 3 else _rnd((M, N), 4, dtype)
        kw = dict(epilogue=_act_code(act), residual=res)
        y, z = _ops().linear16(x, w, b, keep=True, **kw)
        _check_forward(x, w, b, act, res, y, z)
        assert _t().equal(y, _ops().linear16(x, w, b, **kw))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("size", SIZES)
def test_backward(size, dtype):
    M, N, K = size
    for n, act in enumerate(("none", "relu", "gelu", "silu", "sigmoid")):
        say("linear16_backward", size, dtype, act)
        x, w, dy = _rnd((M, K), 1, dtype), _rnd((N, K), 2, dtype, K ** -0.5), _rnd((M, N), 5, dtype)
        z = _rnd((M, N), 6, dtype, 2.0) if act != "none" else None
        pd = _dtype("f32") if n % 2 else None
        dx, dw, db = _ops().linear16_backward(dy, x, w, z, epilogue=_act_code(act), param_dtype=pd)
        assert dx.dtype == x.dtype and dw.dtype == db.dtype == (pd or x.dtype)
        _check_backward(dy, x, w, z, act, dx, dw, db)


def test_parts_of_the_backward_pass():
    """Each gradient alone has the bits that it has among the others."""
    torch, ops = _t(), _ops()
    x, w, dy = _rnd((130, 200), 1, "bf16"), _rnd((264, 200), 2, "bf16"), _rnd((130, 264), 3, "bf16")
    z = _rnd((130, 264), 4, "bf16")
    kw = dict(epilogue=_act_code("gelu"))
    dx, dw, db = ops.linear16_backward(dy, x, w, z, **kw)
    a = ops.linear16_backward(dy, x, w, z, params=False, **kw)
    assert a[1] is None and a[2] is None and torch.equal(a[0], dx)
    a = ops.linear16_backward(dy, x, w, z, input=False, bias=False, **kw)
    assert a[0] is None and a[2] is None and torch.equal(a[1], dw)
    assert ops.linear16_backward(dy, x, w, z, input=False, params=False, **kw) == (None, None, None)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_empty_sizes(dtype):
    torch, ops = _t(), _ops()
    say("linear16 empty")
    x, w, b = _rnd((0, 64), 1, dtype), _rnd((24, 64), 2, dtype), _rnd((24,), 3, dtype)
    assert ops.linear16(x, w, b).shape == (0, 24)
    dx, dw, db = ops.linear16_backward(_rnd((0, 24), 4, dtype), x, w)
    assert dx.shape == (0, 64) and (dw == 0).all() and (db == 0).all()
    # no inputs: the bias alone, and its gradient
    x, w, res, dy = _rnd((130, 0), 1, dtype), _rnd((24, 0), 2, dtype), _rnd((130, 24), 4, dtype), _rnd((130, 24), 5, dtype)
    y = ops.linear16(x, w, b, residual=res)
    assert torch.equal(y, (res.float() + b.float()).to(y.dtype))
    dx, dw, db = ops.linear16_backward(dy, x, w)
    assert dx.shape == (130, 0) and dw.shape == (24, 0)
    _check_backward(dy, x, w, None, "none", None, None, db)
    # no outputs
    x, w = _rnd((130, 64), 1, dtype), _rnd((0, 64), 2, dtype)
    assert ops.linear16(x, w).shape == (130, 0)
    dx, dw, db = ops.linear16_backward(_rnd((130, 0), 4, dtype), x, w)
    assert (dx == 0).all() and dw.shape == (0, 64) and db.shape == (0,)


def _inside(t, lead, tail, value):
    """t's values as a view into a larger matrix of `value` that begins `lead` columns into its rows."""
    torch = _t()
    rows, cols = t.shape
    big = torch.full((rows + 2, cols + lead + tail), value, dtype=t.dtype, device="cuda")
    v = big[1:-1, lead:lead + cols]
    v.copy_(t)
    return big, v


@pytest.mark.parametrize("lead,tail", [(0, 8), (8, 0), (3, 2), (1, 0)])
@pytest.mark.parametrize("size", [(1, 264, 200), (37, 100, 96), (70, 130, 65), (300, 272, 136), (1100, 1032, 264)])
def test_views(size, lead, tail):
    """Operands inside larger matrices of NaN, aligned and not, give the bits of dense copies where the
    alignment is the same kernel's, and results inside others leave those as they were."""
    torch, ops = _t(), _ops()
    M, N, K = size
    say("linear16 views", size, lead, tail)
    nan = float("nan")
    x, w, res, dy = _rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16", K ** -0.5), _rnd((M, N), 3, "bf16"), _rnd((M, N), 4, "bf16")
    b = _rnd((N,), 5, "f32")
    vx, vw, vr, vd = (_inside(t, lead, tail, nan)[1] for t in (x, w, res, dy))
    big, vy = _inside(torch.zeros_like(res), lead, tail, 7.0)
    got, z = ops.linear16(vx, vw, b, epilogue=_act_code("gelu"), residual=vr, keep=True, out=vy)
    assert got is vy
    _check_forward(x, w, b, "gelu", res, vy, z)
    big[1:-1, lead:lead + N] = 7.0
    assert (big == 7).all()
    dx, dw, db = ops.linear16_backward(vd, vx, vw, _inside(z, lead, tail, nan)[1], epilogue=_act_code("gelu"))
    _check_backward(dy, x, w, z, "gelu", dx, dw, db)


def test_residual_in_place():
    torch, ops = _t(), _ops()
    for M, N, K in ((1, 512, 256), (40, 96, 2048), (300, 264, 136), (1030, 1288, 264)):
        x, w, res = _rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16", K ** -0.5), _rnd((M, N), 3, "bf16")
        want = ops.linear16(x, w, residual=res)
        got = ops.linear16(x, w, residual=res, out=res)
        assert got is res and torch.equal(got, want)


def test_leading_dimensions():
    torch, ops = _t(), _ops()
    x, w, res = _rnd((3, 5, 72), 1, "f16"), _rnd((40, 72), 2, "f16"), _rnd((3, 5, 40), 3, "f16")
    y, z = ops.linear16(x, w, residual=res, epilogue=_act_code("silu"), keep=True)
    flat = ops.linear16(x.view(15, 72), w, residual=res.view(15, 40), epilogue=_act_code("silu"))
    assert y.shape == z.shape == (3, 5, 40) and torch.equal(y.view(15, 40), flat)
    dx, dw, db = ops.linear16_backward(res, x, w, z, epilogue=_act_code("silu"))
    assert dx.shape == x.shape
    one = ops.linear16(x[0, 0], w)
    assert one.shape == (40,) and torch.equal(one, ops.linear16(x[0, :1], w)[0])


@pytest.mark.parametrize("size", [(33, 96, 200), (300, 264, 136), (700, 1032, 520)])
def test_infinities_and_nan_stay_in_their_rows(size):
    torch, ops = _t(), _ops()
    M, N, K = size
    x, w, dy = _rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16"), _rnd((M, N), 3, "bf16")
    clean = ops.linear16(x, w)
    x[5, 7], x[M - 1, K - 1] = float("nan"), float("inf")
    y = ops.linear16(x, w)
    bad = torch.zeros(M, dtype=torch.bool, device="cuda")
    bad[5] = bad[M - 1] = True
    assert not torch.isfinite(y[bad]).any() and torch.equal(y[~bad], clean[~bad])
    dx, dw, db = ops.linear16_backward(dy, x, w)
    assert torch.isfinite(dx).all() and torch.isfinite(db).all()
    cols = torch.zeros(K, dtype=torch.bool, device="cuda")
    cols[7] = cols[K - 1] = True
    assert not torch.isfinite(dw[:, cols]).any() and torch.isfinite(dw[:, ~cols]).all()


def test_gradients_against_differences():
    """A layer without activation is linear in x, W and b: differences over any step are exact but for
    the roundings, here sums over a small layer of whole numbers, which have none."""
    torch, ops = _t(), _ops()
    g = torch.Generator(device="cuda").manual_seed(0)

    def ints(*shape):
        return torch.randint(-4, 5, shape, device="cuda", generator=g).to(torch.float16)

    M, N, K = 20, 24, 16
    x, w, b, dy = ints(M, K), ints(N, K), ints(N), ints(M, N)
    dx, dw, db = ops.linear16_backward(dy, x, w, param_dtype=torch.float32)

    def loss(x, w, b):
        return (ops.linear16(x, w, b).double() * dy.double()).sum()

    base = loss(x, w, b)
    for _ in range(4):
        ex, ew, eb = ints(M, K), ints(N, K), ints(N)
        assert loss(x + ex, w, b) - base == (dx.double() * ex.double()).sum()
        assert loss(x, w + ew, b) - base == (dw.double() * ew.double()).sum()
        assert loss(x, w, b + eb) - base == (db.double() * eb.double()).sum()


@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid", "relu"])
def test_slopes_against_differences(act):
    """The formula that the backward pass is held to is the derivative of the forward one's."""
    torch = _t()
    z = torch.linspace(-6, 6, 4001, dtype=torch.float64, device="cuda")[1::2]   # (not 0 itself)
    h = 1e-5
    d = (_act(z + h, act) - _act(z - h, act)) / (2 * h)
    assert float((d - _slope(z, act)).abs().max()) < 1e-8   # h^2 of the third derivative, and 2^-53 / h


def test_the_same_bits_every_time_and_in_a_graph():
    torch, ops = _t(), _ops()
    for M, N, K in ((1, 512, 4096), (48, 200, 4096), (700, 1032, 520)):
        say("linear16 graph", M, N, K)
        x, w, b, res, dy = (_rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16", K ** -0.5), _rnd((N,), 3, "bf16"),
                            _rnd((M, N), 4, "bf16"), _rnd((M, N), 5, "bf16"))
        act = _act_code("gelu")
        ws = torch.empty(max(ops.linear16_workspace_bytes(M, N, K),
                             ops.linear16_backward_workspace_bytes(M, N, K, act), 1), dtype=torch.uint8, device="cuda")

        def step():
            y, z = ops.linear16(x, w, b, epilogue=act, residual=res, keep=True, workspace=ws)
            return (y, z) + ops.linear16_backward(dy, x, w, z, epilogue=act, workspace=ws)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for k in range(3):
            x.copy_(_rnd((M, K), 10 + k, "bf16"))
            dy.copy_(_rnd((M, N), 20 + k, "bf16"))
            want = step()
            torch.cuda.synchronize()
            for t in held:
                t.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, c) for a, c in zip(held, want))
            assert all(torch.equal(a, c) for a, c in zip(step(), want))


def test_two_streams():
    """Calls in flight together on streams of their own, each with its own scratch."""
    torch, ops = _t(), _ops()
    x, w = _rnd((48, 4096), 1, "bf16"), _rnd((200, 4096), 2, "bf16")
    dy = _rnd((48, 200), 3, "bf16")
    want = (ops.linear16(x, w),) + ops.linear16_backward(dy, x, w)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            got.append((ops.linear16(x, w),) + ops.linear16_backward(dy, x, w))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_refusals():
    torch, ops = _t(), _ops()
    x, w, res = _rnd((4, 64), 1, "bf16"), _rnd((8, 64), 2, "bf16"), _rnd((4, 8), 3, "bf16")
    act = _act_code("gelu")

    def refused(f, kind=(ValueError, TypeError, RuntimeError)):
        with pytest.raises(kind):
            f()

    refused(lambda: ops.linear16(x.float(), w), TypeError)
    refused(lambda: ops.linear16(x, w.half()), TypeError)
    refused(lambda: ops.linear16(x, w[:, :60]), ValueError)
    refused(lambda: ops.linear16(x, w.t()), ValueError)
    refused(lambda: ops.linear16(x, w, torch.zeros(7, device="cuda")), ValueError)
    refused(lambda: ops.linear16(x, w, torch.zeros(8, device="cuda", dtype=torch.float16)), TypeError)
    refused(lambda: ops.linear16(x, w, residual=res.float()), TypeError)
    refused(lambda: ops.linear16(x, w, residual=res[:2]), ValueError)
    refused(lambda: ops.linear16(x, w, epilogue=9), RuntimeError)
    refused(lambda: ops.linear16(x, w, out=res.float()), TypeError)
    refused(lambda: ops.linear16(x, w, out=torch.empty(4, 9, device="cuda", dtype=x.dtype)), ValueError)
    refused(lambda: ops.linear16(x, w, workspace=torch.empty(8)), ValueError)
    square = _rnd((64, 64), 4, "bf16")
    refused(lambda: ops.linear16(square, square.clone(), out=square), RuntimeError)
    refused(lambda: ops.linear16(square.clone(), square, out=square), RuntimeError)
    big = _rnd((5, 8), 5, "bf16")
    refused(lambda: ops.linear16(x, w, residual=big[:4], out=big[1:]), RuntimeError)
    refused(lambda: ops.linear16_backward(res, x, w, epilogue=act), ValueError)
    refused(lambda: ops.linear16_backward(res, x, w, res[:, :4], epilogue=act), ValueError)
    refused(lambda: ops.linear16_backward(res[:2], x, w), ValueError)
    refused(lambda: ops.linear16_backward(res.half(), x, w), TypeError)
    refused(lambda: ops.linear16_backward(res, x, w, param_dtype=torch.float64), TypeError)
