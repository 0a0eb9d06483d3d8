"""Layer norm forward and backward against the formula in 64 bits.

Tolerances: a sum of n terms whose longest chain of additions is G has an error of at most
G 2^-24 times the sum of the terms' magnitudes; a row's chain is at most 32 elements in a thread
and 12 levels over threads, the column sums' at most 16 rows of partials, 32 lanes and a
workgroup's own rows.  G = 64 for a row covers the few further roundings of each formula.  The
rounding to the output's type adds half a unit in its last place."""
import numpy as np
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
G = 64


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _ops():
    import cudeep_amd.ops as o
    return o


def _half_ulp(dtype):
    import torch
    return {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]


def _dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _inputs(rows, dim, dtype, pdtype, seed, mean=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, dim, device="cuda", generator=g)
         + mean * torch.randn(rows, 1, device="cuda", generator=g)).to(dtype)
    dy = torch.randn(rows, dim, device="cuda", generator=g).to(dtype)
    w = (1 + 0.3 * torch.randn(dim, device="cuda", generator=g)).to(pdtype)
    b = (0.3 * torch.randn(dim, device="cuda", generator=g)).to(pdtype)
    return x, dy, w, b


def _check(got, ref, bound, dtype, what):
    got = got.double()
    # 2^-24: the least f16 subnormal's half step too
    limit = _half_ulp(dtype) * ref.abs() + bound + 2.0 ** -25
    over = ((got - ref).abs() - limit).max().item() if ref.numel() else -1.0
    assert over <= 0, f"{what}: {over} over its bound"


def _reference(x, dy, w, b, eps):
    """The formula in float64 and the bounds of y, dx, dw, db (dw, db: per column)."""
    import torch
    x, dy = x.double(), dy.double()
    dim = x.shape[1]
    w = torch.ones(dim, device="cuda", dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(dim, device="cuda", dtype=torch.float64) if b is None else b.double()
    mu = x.mean(1, keepdim=True)
    var = ((x - mu) ** 2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    xh = (x - mu) * r
    # xh's own error: the mean's (relative to the mean magnitude) and r's
    exh = G * U * (x.abs().mean(1, keepdim=True) * r + x.abs() * r + xh.abs())
    g = dy * w
    c0, c1 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - c0 - xh * c1)
    m0, m1 = g.abs().mean(1, keepdim=True), (g * xh).abs().mean(1, keepdim=True)
    e1 = G * U * m1 + (g.abs() * exh).mean(1, keepdim=True)
    edx = r * (G * U * (g.abs() + m0 + xh.abs() * m1) + exh * c1.abs() + xh.abs() * e1)
    return {"y": (xh * w + b, exh * w.abs() + G * U * (xh * w).abs() + 4 * U * b.abs()),
            "dx": (dx, edx),
            "dw": ((dy * xh).sum(0), 2 * G * U * (dy * xh).abs().sum(0) + (dy.abs() * exh).sum(0)),
            "db": (dy.sum(0), 2 * G * U * dy.abs().sum(0)),
            "mean": mu[:, 0], "rstd": r[:, 0]}


# widths: each row layout's ends (128, 512, 1024, 2048, 4096, 8192, 16384, 32768), odd ones, one
SHAPES = [(1, 1), (3, 2), (5, 7), (33, 16), (70, 128), (17, 129), (9, 255), (64, 256), (31, 333),
          (40, 512), (21, 513), (1, 1000), (520, 1000), (35, 1024), (11, 1025), (6, 2048),
          (7, 2051), (1, 4096), (130, 4096), (5, 4097), (3, 8191), (4, 8192), (3, 12000),
          (2, 16384), (3, 16385), (2, 32768), (2, 33001), (4099, 40)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_backward(shape, dtype):
    import torch
    ops = _ops()
    rows, dim = shape
    dt = _dtype(dtype)
    pdt = dt if (rows + dim) % 2 else torch.float32
    x, dy, w, b = _inputs(rows, dim, dt, pdt, rows * 7 + dim)
    say("layer norm", shape, dtype, "params", pdt)
    y, mean, rstd = ops.layer_norm(x, w, b, 1e-5, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    torch.cuda.synchronize()
    ref = _reference(x, dy, w, b, 1e-5)
    _check(y, *ref["y"], dt, "y")
    _check(dx, *ref["dx"], dt, "dx")
    _check(dw, *ref["dw"], pdt, "dw")
    _check(db, *ref["db"], pdt, "db")
    assert dw.dtype == pdt and db.dtype == pdt
    scale = x.double().abs().mean(1)
    assert ((mean.double() - ref["mean"]).abs() <= G * U * scale).all()
    assert ((rstd.double() - ref["rstd"]).abs()
            <= G * U * (1 + (scale * ref["rstd"])) * ref["rstd"]).all()
    # without statistics, and once more: the same bits
    assert torch.equal(ops.layer_norm(x, w, b), y)
    for a, c in zip((dx, dw, db), ops.layer_norm_backward(dy, x, mean, rstd, w)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [24, 1000, 20000])
def test_without_parameters(dim, dtype):
    import torch
    ops = _ops()
    dt = _dtype(dtype)
    x, dy, w, b = _inputs(37, dim, dt, dt, dim)
    say("layer norm, no parameters", dim, dtype)
    y, mean, rstd = ops.layer_norm(x, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, params=False)
    assert dw is None and db is None
    ref = _reference(x, dy, None, None, 1e-5)
    _check(y, *ref["y"], dt, "y")
    _check(dx, *ref["dx"], dt, "dx")
    # a bias alone, and gradients of parameters that were one and zero
    _check(ops.layer_norm(x, None, b), *_reference(x, dy, None, b, 1e-5)["y"], dt, "y + b")
    _, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, param_dtype=torch.float32)
    _check(dw, *ref["dw"], torch.float32, "dw")
    _check(db, *ref["db"], torch.float32, "db")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_offsets(dtype):
    """Rows of a wider matrix that begin at odd elements, and outputs the same way; the columns
    beside them stay as they were."""
    import torch
    ops = _ops()
    dt = _dtype(dtype)
    rows, dim = 29, 1003
    x, dy, w, b = _inputs(rows, dim, dt, dt, 5)
    wide = [torch.full((rows, dim + 9), 7.0, device="cuda", dtype=dt) for _ in range(4)]
    views = [t[:, 3:3 + dim] for t in wide]
    views[0].copy_(x)
    views[1].copy_(dy)
    say("layer norm, strided", dtype)
    y, mean, rstd = ops.layer_norm(views[0], w, b, stats=True, out=views[2])
    dx, dw, db = ops.layer_norm_backward(views[1], views[0], mean, rstd, w, out=views[3])
    y2, m2, r2 = ops.layer_norm(x, w, b, stats=True)
    dx2, dw2, db2 = ops.layer_norm_backward(dy, x, m2, r2, w)
    for a, c in ((y, y2), (dx, dx2), (dw, dw2), (db, db2), (mean, m2), (rstd, r2)):
        assert torch.equal(a, c)
    for t in wide:
        assert (t[:, :3] == 7).all() and (t[:, 3 + dim:] == 7).all()


def test_more_than_two_dimensions():
    import torch
    ops = _ops()
    x, dy, w, b = _inputs(30, 64, torch.float32, torch.float32, 2)
    y, mean, rstd = ops.layer_norm(x.view(2, 3, 5, 64), w, b, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy.view(2, 3, 5, 64), x.view(2, 3, 5, 64), mean, rstd, w)
    y2, m2, r2 = ops.layer_norm(x, w, b, stats=True)
    dx2, dw2, db2 = ops.layer_norm_backward(dy, x, m2, r2, w)
    assert y.shape == (2, 3, 5, 64) and torch.equal(y.view(30, 64), y2)
    assert torch.equal(dx.view(30, 64), dx2) and torch.equal(dw, dw2) and torch.equal(db, db2)


def test_no_rows():
    import torch
    ops = _ops()
    x = torch.empty((0, 48), device="cuda")
    w = torch.ones(48, device="cuda")
    y, mean, rstd = ops.layer_norm(x, w, w, stats=True)
    assert y.shape == (0, 48) and mean.numel() == 0
    dx, dw, db = ops.layer_norm_backward(x, x, mean, rstd, w)
    assert dx.shape == (0, 48) and not dw.any() and not db.any()
    dx, dw, db = ops.layer_norm_backward(x.half(), x.half(), mean, rstd)
    assert not dw.any() and not db.any() and dw.dtype == torch.float16


def test_constant_rows_and_large_means():
    """A constant row is exactly zero before the bias (eps alone under the root); a mean 2^12 times the spread
    keeps its digits, as the variance is no difference of squares."""
    import torch
    ops = _ops()
    x = torch.full((4, 512), 3.0, device="cuda")
    assert not ops.layer_norm(x).any()
    g = torch.Generator(device="cuda").manual_seed(3)
    x = 4096 + torch.randn(8, 1536, device="cuda", generator=g)
    ref = _reference(x, x, None, None, 1e-5)
    _check(ops.layer_norm(x), *ref["y"], torch.float32, "y")


def test_faults_stay_in_their_rows():
    import torch
    ops = _ops()
    x, dy, w, b = _inputs(6, 700, torch.float32, torch.float32, 8)
    clean = ops.layer_norm(x, w, b)
    x[1, 5] = float("nan")
    x[4, 699] = float("inf")
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    assert y[1].isnan().all() and y[4].isnan().any()
    keep = [0, 2, 3, 5]
    assert torch.equal(y[keep], clean[keep])
    dx, _, _ = ops.layer_norm_backward(dy, x, mean, rstd, w)
    assert dx[1].isnan().all() and dx[keep].isfinite().all()


@pytest.mark.parametrize("dim", [96, 1000])
def test_gradient_against_differences(dim):
    """Along a random direction v, (L(x + h v) - L(x - h v)) / 2h of the kernel's own forward, L = sum c y,
    against dx . v and the like for w and b.  The difference's own error: its truncation, as the
    64-bit formula has it, and the forward's bound over h."""
    import torch
    ops = _ops()
    rows = 50
    x, c, w, b = _inputs(rows, dim, torch.float32, torch.float32, dim)
    v, _, vw, vb = _inputs(rows, dim, torch.float32, torch.float32, dim + 1)
    h = 2.0 ** -7
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    dx, dw, db = ops.layer_norm_backward(c, x, mean, rstd, w)
    cases = {"x": ((v, None, None), (dx.double() * v.double()).sum(), 0),
             "w": ((None, vw, None), (dw.double() * vw.double()).sum(), 1),
             "b": ((None, None, vb), (db.double() * vb.double()).sum(), 2)}

    def loss(y):
        return (y.double() * c.double()).sum()

    def moved(sign, d):
        return [t if q is None else t + sign * h * q for t, q in zip((x, w, b), d)]

    for name, (d, along, _) in cases.items():
        up, down = moved(1, d), moved(-1, d)
        own = (loss(ops.layer_norm(*up)) - loss(ops.layer_norm(*down))) / (2 * h)
        ends = [_reference(t[0], c, t[1], t[2], 1e-5) for t in (up, down)]
        exact = (loss(ends[0]["y"][0]) - loss(ends[1]["y"][0])) / (2 * h)
        mid = _reference(x, c, w, b, 1e-5)
        slope = {"x": (mid["dx"][0] * v.double()).sum(), "w": (mid["dw"][0] * vw.double()).sum(),
                 "b": (mid["db"][0] * vb.double()).sum()}[name]
        noise = sum(((e["y"][1] + U * e["y"][0].abs()) * c.double().abs()).sum() for e in ends) / (2 * h)
        bound = {"x": ((mid["dx"][1] + U * mid["dx"][0].abs()) * v.double().abs()).sum(),
                 "w": ((mid["dw"][1] + U * mid["dw"][0].abs()) * vw.double().abs()).sum(),
                 "b": ((mid["db"][1] + U * mid["db"][0].abs()) * vb.double().abs()).sum()}[name]
        # the moved inputs are rounded to float32 themselves: U |x| over h, once per end
        step = U / h * {"x": (mid["dx"][0].abs() * (x.double().abs() + h * v.double().abs())).sum(),
                        "w": (mid["dw"][0].abs() * (w.double().abs() + h * vw.double().abs())).sum(),
                        "b": (mid["db"][0].abs() * (b.double().abs() + h * vb.double().abs())).sum()}[name]
        assert abs(own - along) <= abs(exact - slope) + noise + bound + step, name


def test_workspace_stream_and_capture():
    """The caller's workspace and stream, and a captured step replayed between eager work."""
    import torch
    ops = _ops()
    rows, dim = 777, 1000
    x, dy, w, b = _inputs(rows, dim, torch.bfloat16, torch.bfloat16, 11)
    n = ops.layer_norm_backward_workspace_bytes(rows, dim, torch.bfloat16)
    assert n > 0
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")

    def step(x):
        y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
        return (y,) + ops.layer_norm_backward(dy, x, mean, rstd, w, workspace=ws)

    ref = step(x)
    small = torch.empty(n - 1, dtype=torch.uint8, device="cuda")
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    with pytest.raises(Exception, match="workspace"):
        ops.layer_norm_backward(dy, x, mean, rstd, w, workspace=small)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    side.synchronize()
    for a, c in zip(got, ref):
        assert torch.equal(a, c)
    xin = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xin)
    for k in range(4):
        x2 = (x.float() * (1 + 0.5 * k) + k).to(torch.bfloat16)
        xin.copy_(x2)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        for a, c in zip(kept, step(x2)):
            assert torch.equal(a, c), k


def test_rows_beyond_32_bits_of_elements():
    """Offsets over 2^32 bytes and 2^31 elements: the last rows against the same rows alone."""
    import torch
    ops = _ops()
    dim = 4096
    rows = (1 << 31) // dim + 3
    free, _ = torch.cuda.mem_get_info()
    if free < 6 * rows * dim * 2:
        pytest.skip("needs 25 GB of device memory")
    x = torch.zeros((rows, dim), device="cuda", dtype=torch.bfloat16)
    tail, dy, w, b = _inputs(5, dim, torch.bfloat16, torch.bfloat16, 21)
    x[-5:] = tail
    say("layer norm", rows, dim)
    y, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    assert torch.equal(y[-5:], ops.layer_norm(tail, w, b))
    g = torch.zeros_like(x)
    g[-5:] = dy
    dx, dw, db = ops.layer_norm_backward(g, x, mean, rstd, w, out=y)
    t = ops.layer_norm(tail, w, b, stats=True)
    dx2, dw2, db2 = ops.layer_norm_backward(dy, tail, t[1], t[2], w)
    torch.cuda.synchronize()
    assert torch.equal(dx[-5:], dx2)
    # the zero rows add nothing; the five rows meet in another order
    ref = _reference(tail, dy, w, b, 1e-5)
    _check(dw, *ref["dw"], torch.bfloat16, "dw")
    _check(db, *ref["db"], torch.bfloat16, "db")


def test_refusals():
    import torch
    ops = _ops()
    x = torch.randn(4, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    y, mean, rstd = ops.layer_norm(x, w, w, stats=True)
    bad = [lambda: ops.layer_norm(x.cpu()), lambda: ops.layer_norm(x.double()),
           lambda: ops.layer_norm(x.t()), lambda: ops.layer_norm(x[:, :0]),
           lambda: ops.layer_norm(torch.tensor(1.0, device="cuda")),
           lambda: ops.layer_norm(x.view(2, 2, 8).transpose(0, 1)),
           lambda: ops.layer_norm(x[:1].expand(4, 8)),
           lambda: ops.layer_norm(x, w[:7]), lambda: ops.layer_norm(x, w.half()),
           lambda: ops.layer_norm(x.half(), w.half(), w), lambda: ops.layer_norm(x, w.cpu()),
           lambda: ops.layer_norm(x, w, eps=-1.0), lambda: ops.layer_norm(x, w, eps=float("nan")),
           lambda: ops.layer_norm(x, out=x.half()), lambda: ops.layer_norm(x, out=x[:3]),
           lambda: ops.layer_norm_backward(x.half(), x, mean, rstd, w),
           lambda: ops.layer_norm_backward(x[:3], x, mean, rstd, w),
           lambda: ops.layer_norm_backward(x, x, mean[:3], rstd, w),
           lambda: ops.layer_norm_backward(x, x, mean.double(), rstd, w),
           lambda: ops.layer_norm_backward(x, x, mean, rstd, w, param_dtype=torch.float16),
           lambda: ops.layer_norm_backward(x, x, mean, rstd, param_dtype=torch.float64)]
    for k, f in enumerate(bad):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            f()
            pytest.fail(f"refusal {k} was accepted")
