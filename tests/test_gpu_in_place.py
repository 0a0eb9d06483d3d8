"""Row operators whose result takes the place of an input: the same bits as into a tensor of its
own, on either side of the widths at which the kernels change (8192: the parameters' sums; 16384
and 32768: rows that no longer stay in registers)."""
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _dtype(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _normal(shape, seed, dtype):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) + 0.5).to(dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [100, 1000, 4096, 8192, 8193, 12000, 16384, 20000])
def test_layer_norm_backward(dim, dtype):
    """70 rows: the column sums of wide rows come from three parts."""
    import torch
    from cudeep_amd import ops
    dt = _dtype(dtype)
    x, dy = _normal((70, dim), dim, dt), _normal((70, dim), dim + 1, dt)
    w = _normal((dim,), 3, dt)
    say("layer norm backward in place", dim, dtype)
    _, mean, rstd = ops.layer_norm(x, w, stats=True)
    want = ops.layer_norm_backward(dy, x, mean, rstd, w)
    for name in ("dy", "x"):
        gx, gy = x.clone(), dy.clone()
        out = gx if name == "x" else gy
        got = ops.layer_norm_backward(gy, gx, mean, rstd, w, out=out)
        assert got[0] is out
        for part, a, b in zip(("dx", "dw", "db"), got, want):
            assert torch.equal(a, b), (name, part)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [100, 4096, 16384, 33001])
def test_layer_norm(dim, dtype):
    import torch
    from cudeep_amd import ops
    dt = _dtype(dtype)
    x, w = _normal((9, dim), dim, dt), _normal((dim,), 3, dt)
    say("layer norm in place", dim, dtype)
    want = ops.layer_norm(x, w, w)
    assert torch.equal(ops.layer_norm(x, w, w, out=x), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_activation(dtype):
    import torch
    from cudeep_amd import _lib as L
    from cudeep_amd import ops
    dt = _dtype(dtype)
    z, dy = _normal((33, 1000), 5, dt), _normal((33, 1000), 6, dt)
    say("activation8 in place", dtype)
    y, kept = ops.activation8(z, L.EPI_GELU)
    dz = ops.activation_backward8(dy, kept, L.EPI_GELU)
    y2, kept2 = ops.activation8(z, L.EPI_GELU, out=z)
    assert y2 is z and torch.equal(y2, y)
    assert torch.equal(kept2.q.view(torch.uint8), kept.q.view(torch.uint8))
    assert torch.equal(kept2.scale.view(torch.uint8), kept.scale.view(torch.uint8))
    assert torch.equal(ops.activation_backward8(dy, kept, L.EPI_GELU, out=dy), dz)
