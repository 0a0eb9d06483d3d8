"""Rows so wide that one workgroup for each of their parts would be 2^32 threads and more, which a
launch does not hold."""
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()
    import torch
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")


def test_quantize_tiles():
    """Two launches of 2^28 columns and one of the rest."""
    import torch
    from cudeep_amd import ops
    cols = (1 << 29) + 300
    x = torch.zeros((2, cols), device="cuda", dtype=torch.bfloat16)
    at = [0, 5, (1 << 28) - 1, 1 << 28, (1 << 28) + 129, (1 << 29) - 1, 1 << 29, cols - 1]
    g = torch.Generator(device="cuda").manual_seed(1)
    x[:, at] = torch.randn((2, len(at)), device="cuda", generator=g).to(torch.bfloat16)
    for dt in (torch.float8_e8m0fnu, torch.float32):
        say("quantize8 tiles", cols, dt)
        b = ops.quantize8(x, 128, scale_dtype=dt)
        parts = [(c // 128 * 128, min(c // 128 * 128 + 128, cols)) for c in at]
        for lo, hi in parts:
            want = ops.quantize8(x[:, lo:hi], 128, scale_dtype=dt)
            assert torch.equal(b.q[:, lo:hi].view(torch.uint8), want.q.view(torch.uint8))
            assert b.scale[0, lo // 128].float() == want.scale[0, 0].float()
        assert int(b.q.view(torch.uint8).count_nonzero()) <= 2 * len(at)
        one = 127 if dt == torch.float8_e8m0fnu else 1.0
        plain = b.scale.view(torch.uint8) if dt == torch.float8_e8m0fnu else b.scale
        assert int((plain != one).sum()) <= len(at)
        del b, plain


def test_layer_norm_backward():
    """2^27 + 64 columns: the parameters' gradients of two rows, which are exact products rounded."""
    import torch
    from cudeep_amd import ops
    dim = (1 << 27) + 64
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((2, dim), device="cuda", dtype=torch.bfloat16, generator=g)
    dy = torch.randint(-4, 5, (2, dim), device="cuda", generator=g).to(torch.bfloat16)
    say("layer norm backward", dim)
    y, mean, rstd = ops.layer_norm(x, stats=True)
    dx, dw, db = ops.layer_norm_backward(dy, x, mean, rstd, param_dtype=torch.float32)
    for part in (slice(0, 1 << 16), slice(dim - (1 << 16), dim), slice(dim // 2, dim // 2 + (1 << 16))):
        xh = (x[:, part].double() - mean.double()[:, None]) * rstd.double()[:, None]
        t = dy[:, part].double() * xh
        # xh: two roundings and that of the difference; one of the product, one of the sum
        assert ((dw[part].double() - t.sum(0)).abs() <= 5 * 2.0 ** -24 * t.abs().sum(0)
                + 2.0 ** -24 * (dy[:, part].double().abs() * mean.double().abs()[:, None] * rstd.double()[:, None]).sum(0)).all()
        assert torch.equal(db[part].double(), dy[:, part].double().sum(0))
        assert ((y[:, part].double() - xh).abs() <= 2.0 ** -8 * xh.abs() + 2.0 ** -25).all()
    assert dx.isfinite().all()
