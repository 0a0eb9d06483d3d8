"""Gradients and masks at the ends of the ranges that calls allow: the entropy's gradient at a low temperature,
large and over masked logits, and long rows whose first part is masked with the type's lowest value.  Bounds
as in test_gpu_logits.py."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_logits import _check_backward, _check_logprobs, _ints, _logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("temperature,h", [(1e-6, 1000.0), (1e-3, 1e6), (1.0, 1e9), (1e6, 1e9)])
def test_large_gradients_of_the_entropy_over_masks(temperature, h, dtype):
    import torch
    from cudeep_amd import ops
    say("entropy's gradient", temperature, h, dtype)
    x, t = _logits(8, 900, 1, dtype, 3.0 * min(temperature, 1.0)), _ints(0, 900, (8,), 2)
    x[0::4, ::2], x[1::4, ::2] = -float("inf"), torch.finfo(x.dtype).min
    x[2, 1:] = -float("inf")
    r = ops.token_logprobs(x, t, entropy=True, temperature=temperature)
    e = _check_logprobs(x, t, temperature, r, 0)
    gh = torch.full((8,), h, device="cuda")
    dx = ops.token_logprobs_backward(None, x, t, r.stats, entropy=r.entropy, grad_entropy=gh, temperature=temperature)
    assert torch.isfinite(dx.float()).all()
    _check_backward(x, t, e, None, gh, dx)


@pytest.mark.parametrize("temperature", [1e-6, 1.0, 1e6])
@pytest.mark.parametrize("rows", [1, 600])
def test_rows_that_begin_with_the_lowest_value(rows, temperature):
    import torch
    from cudeep_amd import ops
    vocab = 400001 if rows == 1 else 20001
    say("lowest values first", rows, temperature)
    x = torch.full((rows, vocab), torch.finfo(torch.float32).min, device="cuda")
    x[:, -1], x[:, -2] = 1.0, 1.0
    t = torch.full((rows,), vocab - 1, device="cuda")
    r = ops.token_logprobs(x, t, entropy=True, top=2, temperature=temperature)
    assert _check_logprobs(x, t, temperature, r, 2)
