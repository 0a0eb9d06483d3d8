"""Results that lie beside their inputs in one buffer, without sharing a byte, are no overlap."""
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("rows", [1, 9])
@pytest.mark.parametrize("first", [True, False])
def test_columns_beside_each_other(rows, first):
    import torch
    from cudeep_amd import _lib as L
    from cudeep_amd import ops
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, 64, device="cuda", generator=g)
    w = ops.quantize8(torch.randn(64, 64, device="cuda", generator=g), 128)
    buf = torch.zeros(rows, 128, device="cuda")
    a, b = (buf[:, :64], buf[:, 64:]) if first else (buf[:, 64:], buf[:, :64])
    say("results beside inputs", rows, first)
    _, kept = ops.activation8(x, L.EPI_GELU)
    _, mean, rstd = ops.layer_norm(x, stats=True)
    for f in (lambda t, out: ops.layer_norm(t, out=out), lambda t, out: ops.linear8(t, w, out=out),
              lambda t, out: ops.layer_norm_backward(t, x, mean, rstd, params=False, out=out)[0],
              lambda t, out: ops.activation8(t, L.EPI_GELU, out=out)[0],
              lambda t, out: ops.activation_backward8(t, kept, L.EPI_GELU, out=out)):
        want = f(x, None)
        a.copy_(x)
        assert torch.equal(f(a, b), want) and torch.equal(a, x)
    # and rows after rows
    two = torch.zeros(2 * rows, 64, device="cuda")
    two[:rows] = x
    assert torch.equal(ops.linear8(two[:rows], w, out=two[rows:]), ops.linear8(x, w))


def test_refusals():
    import torch
    from cudeep_amd import ops
    x = torch.zeros(9, 64, device="cuda")
    w = ops.quantize8(torch.zeros(64, 64, device="cuda"), 128)
    for f in (lambda: ops.linear8(x, w, out=x), lambda: ops.linear8(x[:8], w, out=x[1:]),
              lambda: ops.layer_norm(x[:8], out=x[1:])):
        with pytest.raises(RuntimeError, match="overlap"):
            f()
