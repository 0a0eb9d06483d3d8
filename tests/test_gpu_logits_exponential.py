"""The exponential of float32 logits.  A row of one 0 and values down to -85 has the sum 1 (the rest is below 2^-30) and
L = 0, so that l is the logit itself and a gradient is weight exp(x), with no other rounding in its exponent.

Bound.  The exponential's argument in base 2 is a product and its rest, known to 2^-48 of it; the hardware's power of two is
off by 2^-22; the factor 1 + rest and the two products after it by 2^-24 each; L by less than 2^-30."""
import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu

BOUND = 2.0 ** -22 + 4 * 2.0 ** -24 + 2.0 ** -30


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("rows,pad", [(3, 0), (600, 0), (2, 70000)])   # one workgroup a row, and rows in parts
@pytest.mark.parametrize("temperature", [1.0, 0.5, 4.0])              # (exact scales)
def test_gradients(rows, pad, temperature):
    import torch
    from cudeep_amd import ops
    say("exponential", rows, pad, temperature)
    values = -torch.arange(25 * 16, 85 * 16, device="cuda", dtype=torch.float32) / 16 * temperature
    x = torch.full((rows, 1 + len(values) + pad), -float("inf"), device="cuda")
    x[:, 0], x[:, 1:1 + len(values)] = 0.0, values
    want = torch.exp(values.double() / temperature) / temperature
    one, t = torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.int64, device="cuda")
    r = ops.token_logprobs(x, t, temperature=temperature)
    assert (r.stats == 0).logical_or(r.stats.abs() < 2.0 ** -30).all() and (r.logprob.abs() < 2.0 ** -30).all()
    dx = ops.token_logprobs_backward(one, x, t, r.stats, temperature=temperature)
    loss, grad = ops.distill_loss(x, t[:, None], torch.ones(rows, 1, device="cuda"), temperature=temperature, weight=one)
    for got, sign in ((dx, -1.0), (grad, 1.0)):
        off = (got[:, 1:1 + len(values)].double() * sign / want - 1).abs().max()
        assert float(off) < BOUND, float(off) * 2 ** 24
        assert (got[:, 1 + len(values):] == 0).all()
