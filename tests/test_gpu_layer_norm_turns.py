"""Layer norm where a workgroup walks several rows: at least three turns in the backward pass, the last
one ragged, of every row layout, with data in every row.  Formula and bounds as in
test_gpu_layer_norm.py; a column's chain is at most 5 turns, 32 rows of a workgroup side by side, 32
partials of a lane and 16 lanes, 85 additions of the 128 that the bound holds."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_layer_norm import _check, _dtype, _inputs, _reference

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


# (rows, dim): rows side by side in a workgroup, its workgroups at most
SHAPES = {(40001, 100): (32, 512), (12301, 300): (8, 512), (4099, 1000): (4, 512), (3001, 2048): (2, 512),
          (1100, 4096): (1, 512), (1100, 4001): (1, 512), (600, 8192): (1, 256), (600, 8000): (1, 256)}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", list(SHAPES))
def test_backward(shape, dtype):
    import torch
    from cudeep_amd import ops
    rows, dim = shape
    side, groups = SHAPES[shape]
    dt = _dtype(dtype)
    assert ops.layer_norm_backward_workspace_bytes(rows, dim, dt) == groups * 2 * dim * 4
    assert rows > 2 * groups * side and rows % (groups * side)
    pdt = dt if dim % 2 == 0 else torch.float32
    x, dy, w, b = _inputs(rows, dim, dt, pdt, rows + dim)
    say("layer norm backward, several turns", shape, dtype)
    _, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    ref = _reference(x, dy, w, b, 1e-5)
    _check(dx, *ref["dx"], dt, "dx")
    _check(dw, *ref["dw"], pdt, "dw")
    _check(db, *ref["db"], pdt, "db")
    for a, c in zip((dx, dw, db), ops.layer_norm_backward(dy, x, mean, rstd, w)):
        assert torch.equal(a, c)
    # in place, without parameters' gradients and without a weight
    assert torch.equal(ops.layer_norm_backward(dy, x, mean, rstd, w, params=False)[0], dx)
    one = ops.layer_norm_backward(dy, x, mean, rstd)[0]
    assert torch.equal(ops.layer_norm_backward(dy.clone(), x, mean, rstd, torch.ones_like(w))[0], one)
    gy = dy.clone()
    for a, c in zip(ops.layer_norm_backward(gy, x, mean, rstd, w, out=gy), (dx, dw, db)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(600, 8200), (600, 16384), (601, 20000)])
def test_wide_rows(shape, dtype):
    """Column sums apart: 19 parts of 32 rows."""
    from cudeep_amd import ops
    rows, dim = shape
    dt = _dtype(dtype)
    x, dy, w, b = _inputs(rows, dim, dt, dt, rows + dim)
    assert ops.layer_norm_backward_workspace_bytes(rows, dim, dt) == 19 * 2 * dim * 4
    say("layer norm backward, wide rows", shape, dtype)
    _, mean, rstd = ops.layer_norm(x, w, b, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, w)
    ref = _reference(x, dy, w, b, 1e-5)
    _check(dx, *ref["dx"], dt, "dx")
    _check(dw, *ref["dw"], dt, "dw")
    _check(db, *ref["db"], dt, "db")


@pytest.mark.parametrize("rows,dim", [((1 << 24) + 5, 8), ((1 << 20) + 3, 2049)])
def test_forward(rows, dim):
    """More rows than one walk of the largest grid: the same bits as each half alone."""
    import torch
    from cudeep_amd import ops
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("needs 20 GB of device memory")
    g = torch.Generator(device="cuda").manual_seed(dim)
    x = torch.randn((rows, dim), device="cuda", dtype=torch.bfloat16, generator=g)
    w = torch.randn(dim, device="cuda", generator=g)
    say("layer norm, more rows than the grid", rows, dim)
    y, mean, rstd = ops.layer_norm(x, w, w, stats=True)
    for part in (slice(0, rows // 2), slice(rows // 2, rows)):
        got = ops.layer_norm(x[part], w, w, stats=True)
        for a, c in zip(got, (y[part], mean[part], rstd[part])):
            assert torch.equal(a, c)
