"""Gradients of the activations at values whose square overflows fp32: the slopes there are 0, 1
(or, of LeakyReLU, alpha), to the last bit."""
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu", "sigmoid", "tanh", "leaky"])
def test_slopes(act, dtype):
    """One value a row, so that each has a scale of its own; the last ones round to 2^128 in 8 bits."""
    import torch
    from cudeep_amd import _lib as L
    from cudeep_amd import ops
    code = {"relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU, "sigmoid": L.EPI_SIGMOID,
            "tanh": L.ACT_TANH, "leaky": L.ACT_LEAKY_RELU}[act]
    large = [1e6, 1e13, 1.8e19, 1.9e19, 1e25, 1e38, 3.2e38, 3.4e38]
    z = torch.tensor(large + [-v for v in large], device="cuda").view(-1, 1)
    dt = getattr(torch, dtype)
    say("activation8 large values", act, dtype)
    _, kept = ops.activation8(z, code, alpha=0.25)
    dz = ops.activation_backward8(torch.full_like(z, 3.0, dtype=dt), kept, code, alpha=0.25)
    up, down = {"relu": (1, 0), "gelu": (1, 0), "silu": (1, 0), "sigmoid": (0, 0), "tanh": (0, 0),
                "leaky": (1, 0.25)}[act]
    n = len(large)
    assert (dz[:n].float() == 3.0 * up).all(), dz[:n].view(-1).tolist()
    assert (dz[n:].float() == 3.0 * down).all(), dz[n:].view(-1).tolist()


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_values(act):
    """The values themselves: z above, 0 below."""
    import torch
    from cudeep_amd import _lib as L
    from cudeep_amd import ops
    code = {"gelu": L.EPI_GELU, "silu": L.EPI_SILU}[act]
    for dt in (torch.float32, torch.bfloat16):
        z = torch.tensor([[1e13, 1.9e19, 1e38, -1e13, -1.9e19, -1e38]], device="cuda").to(dt)
        y, _ = ops.activation8(z, code)
        assert torch.equal(y[0, :3], z[0, :3]) and not y[0, 3:].any()
