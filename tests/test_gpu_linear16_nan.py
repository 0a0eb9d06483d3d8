"""NaN and infinities through each epilogue of the 16-bit Linear layer, in each kind of kernel: a NaN in a row or a
weight shows in everything that the formula has it in, and in nothing else."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.routes16 import linear16_kernel
from tests.test_gpu_linear16 import _act, _act_code, _rnd

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "gelu", "silu", "sigmoid"]
NAN, INF = float("nan"), float("inf")
# (kernel, in slices, M, N, K)
CASES = [("direct", False, 33, 96, 200), ("any", False, 70, 130, 65), ("ring 64", False, 300, 264, 136),
         ("ring 64", True, 136, 264, 4136), ("any", True, 299, 203, 1777), ("tall", False, 1304, 1288, 200),
         ("ring 128", False, 1400, 1608, 264), ("tile 128", False, 2104, 2184, 200), ("turns", False, 3600, 3592, 200),
         ("any 128", False, 1801, 1807, 93)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", CASES)
def test_forward(case, dtype):
    import torch
    from cudeep_amd import ops
    name, slices, M, N, K = case
    got = linear16_kernel("forward", M, N, K, K % 8 == 0)
    assert got[0] == name and (got[1] > 1) == slices
    for act in ACTS:
        say("nan", case, dtype, act)
        x, w, res = _rnd((M, K), 1, dtype), _rnd((N, K), 2, dtype, K ** -0.5), _rnd((M, N), 3, dtype)
        kw = dict(epilogue=_act_code(act), residual=res, keep=True)
        clean, zclean = ops.linear16(x, w, **kw)
        x[5, 7], w[3, 2], x[M - 1, K - 1] = NAN, NAN, INF
        y, z = ops.linear16(x, w, **kw)
        bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
        bad[5], bad[:, 3] = True, True
        assert torch.isnan(y[bad]).all() and torch.isnan(z[bad]).all()
        last = torch.zeros_like(bad)
        last[M - 1] = True
        other = ~bad & ~last
        assert torch.equal(y[other], clean[other]) and torch.equal(z[other], zclean[other])
        # the infinite row, by the formula in 64 bits
        side = ~bad[M - 1]
        zx = (torch.sign(w[side, K - 1].double()) * INF).to(z.dtype)
        assert torch.equal(z[M - 1][side], zx)
        want = _act(zx.double(), act) + res[M - 1][side].double()
        row = y[M - 1][side].double()
        assert torch.equal(torch.isnan(row), torch.isnan(want)) and torch.equal(row[torch.isinf(want)], want[torch.isinf(want)])
        assert torch.equal(torch.isfinite(row), torch.isfinite(want))


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_slopes(dtype, bias):
    """Through a weight of ones on its diagonal the input's gradient is dz itself."""
    import torch
    from cudeep_amd import ops
    M, N = 40, 72
    w, x, g = torch.eye(N, device="cuda").to(_rnd((1,), 1, dtype).dtype), _rnd((M, N), 2, dtype), _rnd((M, N), 3, dtype)
    for act in ACTS[1:]:
        say("slopes", dtype, act)
        z = _rnd((M, N), 4, dtype)
        kw = dict(epilogue=_act_code(act), bias=bias)
        clean = ops.linear16_backward(g, x, w, z, **kw)[0]
        z[3, 5], z[7, 9], z[9, 11], z[11, 13] = NAN, INF, -INF, -0.0
        dx, dw, db = ops.linear16_backward(g, x, w, z, **kw)
        same = torch.ones((M, N), dtype=torch.bool, device="cuda")
        same[3], same[7, 9], same[9, 11], same[11, 13] = False, False, False, False
        assert torch.equal(dx[same], clean[same])
        assert dx[7, 9] == (0 if act == "sigmoid" else g[7, 9]) and dx[9, 11] == 0
        if act == "relu":
            assert torch.equal(dx[3, 6:], clean[3, 6:]) and dx[3, 5] == g[3, 5] and dx[11, 13] == 0
        else:
            assert torch.isnan(dx[3]).all() and torch.isnan(dw[5]).all() and torch.isfinite(dw[6:]).all()
            assert not bias or torch.isnan(db[5])
