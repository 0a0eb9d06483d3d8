"""The bias gradient of the 16-bit Linear layer behind an activation: the column sums of dz = grad epi'(z) in
float32, before dz is rounded to 16 bits for the products.

Bound.  The slope is off by 2^-20 of 1 + |z| (the hardware's exponential and reciprocal), times grad; a float32
sum of M values in any order by (M + 8) 2^-24 of the sum of their magnitudes.  A 16-bit result is off by half
a step of its own."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_linear16 import U, _act_code, _dtype, _inside, _rnd, _slope, _within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _check(dy, z, act, db):
    M = dy.shape[0]
    g = dy.double()
    dz = g * _slope(z.double(), act)
    e = 2.0 ** -20 * g.abs() * (1 + z.double().abs())
    _within(db, dz.sum(0), e.sum(0) + (M + 8) * U * (dz.abs() + e).sum(0), "db")


# one row; columns of no whole 8, and more than a workgroup's 256; rows of no whole 32; parts of several rounds; one
# part; operands past 64 MB; outputs without inputs
SIZES = [(1, 1, 8), (1, 300, 64), (7, 9, 16), (33, 257, 24), (64, 256, 40), (513, 1031, 72), (8192, 256, 64),
         (20001, 24, 8), (4097, 513, 16), (40, 300000, 8), (8200, 4104, 8), (130, 24, 0)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("size", SIZES)
def test_bias_gradient(size, dtype):
    import torch
    from cudeep_amd import ops
    M, N, K = size
    x, w, dy, z = _rnd((M, K), 1, dtype), _rnd((N, K), 2, dtype), _rnd((M, N), 3, dtype), _rnd((M, N), 4, dtype, 2.0)
    for act in ("gelu", "silu", "sigmoid", "relu"):
        for pd in (torch.float32, None):
            say("bias gradient", size, dtype, act, pd)
            kw = dict(epilogue=_act_code(act), param_dtype=pd)
            dx, dw, db = ops.linear16_backward(dy, x, w, z, **kw)
            _check(dy, z, act, db)
            # the products' gradients do not depend on whether the bias has one
            alone = ops.linear16_backward(dy, x, w, z, bias=False, **kw)
            assert torch.equal(alone[0], dx) and torch.equal(alone[1], dw) and alone[2] is None
            none, same, sums = ops.linear16_backward(dy, x, w, z, input=False, **kw)
            assert none is None and torch.equal(same, dw) and torch.equal(sums, db)


@pytest.mark.parametrize("lead,tail", [(8, 8), (3, 2)])
def test_views(lead, tail):
    import torch
    from cudeep_amd import ops
    M, N, K = 300, 517, 40
    x, w, dy, z = _rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16"), _rnd((M, N), 3, "bf16"), _rnd((M, N), 4, "bf16")
    vd, vz = (_inside(t, lead, tail, float("nan"))[1] for t in (dy, z))
    db = ops.linear16_backward(vd, x, w, vz, epilogue=_act_code("silu"), param_dtype=torch.float32)[2]
    _check(dy, z, "silu", db)


def test_values_whose_slope_passes_the_type():
    """GELU's slope is up to 1.13: dz past float16's largest value is infinite as an operand, the bias's
    gradient, in float32, is not; an infinite and a NaN gradient stay in their columns."""
    import torch
    from cudeep_amd import ops
    M, N, K = 40, 48, 16
    x, w, dy, z = _rnd((M, K), 1, "f16"), _rnd((N, K), 2, "f16"), _rnd((M, N), 3, "f16"), _rnd((M, N), 4, "f16")
    dy[3], z[3] = 65504.0, 1.5
    kw = dict(epilogue=_act_code("gelu"), param_dtype=torch.float32)
    db = ops.linear16_backward(dy, x, w, z, **kw)[2]
    assert torch.isfinite(db).all()
    _check(dy, z, "gelu", db)
    dy[5, 7], dy[6, 9], z[8, 11] = float("nan"), float("inf"), float("nan")
    db = ops.linear16_backward(dy, x, w, z, **kw)[2]
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    keep[[7, 9, 11]] = False
    assert not torch.isfinite(db[~keep]).any()
    _check(dy[:, keep], z[:, keep], "gelu", db[keep])


def test_in_a_graph():
    import torch
    from cudeep_amd import ops
    M, N, K = 700, 1032, 136
    act = _act_code("gelu")
    x, w, dy, z = _rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16"), _rnd((M, N), 3, "bf16"), _rnd((M, N), 4, "bf16")
    ws = torch.empty(ops.linear16_backward_workspace_bytes(M, N, K, act), dtype=torch.uint8, device="cuda")

    def step():
        return ops.linear16_backward(dy, x, w, z, epilogue=act, param_dtype=_dtype("f32"), workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        dy.copy_(_rnd((M, N), 20 + k, "bf16"))
        want = step()
        torch.cuda.synchronize()
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        _check(dy, z, "gelu", held[2])
