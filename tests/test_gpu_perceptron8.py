"""The operators together: layer norm, 8-bit checkpoints and 8-bit products in one perceptron.

Gradients are compared with 64-bit formulas on the values that the checkpoints hold.  Sums of n
terms in fp32 stray at most n 2^-24 of the sum of magnitudes; along the chain of at most four such
sums (a row's of hidden terms, a column's of `rows`) every term's own error adds.  Relative to the
Frobenius norm of the sums of magnitudes that is at most (rows + 2 hidden + 2 dim) 2^-24 and 64
roundings of single steps (activation slopes, layer norm)."""
import pytest

from tests.gpu_util import require_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _restored(b):
    from cudeep_amd import ops
    return ops.dequantize8(b).double().cpu()


@pytest.mark.parametrize("rows,dim,hidden", [(1, 128, 256), (300, 200, 333), (256, 256, 512)])
def test_gradients(rows, dim, hidden):
    import torch
    from cudeep_amd.examples.perceptron8 import Perceptron8
    torch.manual_seed(rows + dim)
    model = Perceptron8(dim, hidden, dtype=torch.float32)
    x = torch.randn(rows, dim, device="cuda")
    dout = torch.randn(rows, dim, device="cuda")
    out, kept = model.forward(x)
    dx, grads = model.backward(dout, kept)
    h8, z8, y8 = (_restored(b) for b in kept[3:])
    w1, w2, g64, x64 = (t.double().cpu() for t in (model.w1, model.w2, dout, x))

    def slope(v):
        v = v.clone().requires_grad_(True)
        torch.nn.functional.gelu(v, approximate="tanh").sum().backward()
        return v.grad

    s = slope(z8)
    dy, mag_y = g64 @ w2, g64.abs() @ w2.abs()
    dz, mag_z = dy * s, mag_y * (s.abs() + 1)
    dh, mag_h = dz @ w1, mag_z @ w1.abs()
    xv = x64.clone().requires_grad_(True)
    gain = model.gain.double().cpu().requires_grad_(True)
    shift = model.shift.double().cpu().requires_grad_(True)
    (torch.nn.functional.layer_norm(xv, (dim,), gain, shift) * dh).sum().backward()
    xh = (x64 - x64.mean(1, keepdim=True)) / (x64.var(1, keepdim=True, unbiased=False) + 1e-5).sqrt()
    rstd = 1 / (x64.var(1, keepdim=True, unbiased=False) + 1e-5).sqrt()
    mag_x = rstd * (mag_h + mag_h.mean(1, keepdim=True) + xh.abs() * (mag_h * xh.abs()).mean(1, keepdim=True))
    tol = (rows + 2 * hidden + 2 * dim + 64) * 2.0 ** -24
    for name, got, want, mag in (
            ("w2", grads["w2"], g64.T @ y8, g64.abs().T @ y8.abs()),
            ("b2", grads["b2"], g64.sum(0), g64.abs().sum(0)),
            ("w1", grads["w1"], dz.T @ h8, mag_z.T @ h8.abs()),
            ("b1", grads["b1"], dz.sum(0), mag_z.sum(0)),
            ("gain", grads["gain"], gain.grad, (mag_h * xh.abs()).sum(0)),
            ("shift", grads["shift"], shift.grad, mag_h.sum(0)),
            ("x", dx, xv.grad + g64, mag_x + g64.abs())):
        err = (got.double().cpu() - want).norm() / mag.norm()
        assert err <= tol, (name, float(err), tol)


@pytest.mark.parametrize("name", ["float32", "bfloat16", "float16"])
def test_training_and_inference(name):
    """The loss falls, and inference in 8 bits stays within what its roundings can do: each of
    the four operands is off by at most 2^-4 of itself, sums of random signs average it."""
    import torch
    from cudeep_amd.examples.perceptron8 import Perceptron8, train
    torch.manual_seed(3)
    dtype = getattr(torch, name)
    x = torch.randn(512, 256, device="cuda").to(dtype)
    target = x + torch.sin(3.0 * x.float()).to(dtype)
    model = Perceptron8(256, 512, dtype=dtype)
    losses = train(model, x, target, steps=30, rate=4.0)   # (20 diverges in 64 bits too)
    assert losses[-1] < 0.9 * losses[0]
    out, kept = model.forward(x)
    assert all(b.q.element_size() == 1 for b in kept[3:])
    near = model.infer(x, model.quantised())
    assert near.dtype == dtype
    assert (near.float() - out.float()).norm() <= 2.0 ** -3 * (out.float() - x.float()).norm()
