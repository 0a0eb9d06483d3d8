"""The kernels that read logits, each with every number of threads it is built for, and gradients that pass the
caches by, in place and beside their logits.  Bounds as in test_gpu_logits.py."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_logits import _check_backward, _check_distill, _check_logprobs, _ints, _logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(255, 40009), (257, 75001), (511, 40009), (513, 40009), (513, 39999), (127, 70001), (128, 70001)])
def test_logprobs_and_gradient(size, dtype):
    import torch
    from cudeep_amd import ops
    rows, vocab = size
    say("token_logprobs", size, dtype)
    x, t = _logits(rows, vocab, 1, dtype), _ints(0, vocab, (rows,), 2)
    x[::9, ::3] = -float("inf")
    for top, entropy in ((0, True), (0, False), (7, False)):
        r = ops.token_logprobs(x, t, entropy=entropy, top=top, temperature=1.3)
        e = _check_logprobs(x, t, 1.3, r, top)
    g = torch.randn(rows, device="cuda")
    r = ops.token_logprobs(x, t, entropy=True, temperature=1.3)
    dx = ops.token_logprobs_backward(g, x, t, r.stats, entropy=r.entropy, grad_entropy=g, temperature=1.3)
    _check_backward(x, t, e, g, g, dx)
    same = ops.token_logprobs_backward(g, x, t, r.stats, entropy=r.entropy, grad_entropy=g, temperature=1.3, out=x)
    assert same is x and torch.equal(x, dx)


@pytest.mark.parametrize("size", [(513, 33001, "f32"), (513, 64003, "bf16"), (600, 24001, "bf16"), (1500, 24001, "f16"),
                                  (2801, 12001, "f16"), (2801, 5999, "f32"), (127, 70001, "f16"), (128, 70001, "f32"),
                                  (511, 64003, "f16")])
def test_distill(size):
    import torch
    from cudeep_amd import ops
    rows, vocab, dtype = size
    say("distill_loss", size)
    x = _logits(rows, vocab, 1, dtype)
    idx, val, w = _ints(0, vocab, (rows, 20), 2), torch.randn(rows, 20, device="cuda"), torch.rand(rows, device="cuda")
    idx[::4, 5:] = -1
    loss, grad = ops.distill_loss(x, idx, val, weight=w, temperature=2.0)
    _check_distill(x, idx, val, 2.0, w, loss, grad)
    assert torch.equal(ops.distill_loss(x, idx, val, temperature=2.0), loss)
    again, same = ops.distill_loss(x, idx, val, weight=w, temperature=2.0, out=x)
    assert same is x and torch.equal(again, loss) and torch.equal(x, grad)
