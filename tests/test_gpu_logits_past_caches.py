"""Gradients of logits that pass the caches by, in part or whole, with every number of threads, beside their logits and
in their place, and a head's products that read them next.  Bounds as in test_gpu_logits.py."""
import ctypes

import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_logits import _check_backward, _check_distill, _check_logprobs, _ints, _logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _past(rows, vocab, dtype):
    from cudeep_amd import _lib as L
    f = L.lib().cdxi_logits_past_caches
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    return f(rows, vocab, {"f32": 0, "f16": 2, "bf16": 3}[dtype])


# rows, vocabulary, type, what passes: rows of less than 48 KB (256 threads), 128 KB (512) and more (1024)
@pytest.mark.parametrize("size", [(2801, 12001, "f16", 1), (9001, 12001, "bf16", 2), (1500, 24001, "bf16", 1),
                                  (4300, 24001, "f16", 2), (513, 64003, "f16", 1), (1600, 64003, "bf16", 2),
                                  (2801, 5999, "f32", 2), (1001, 16411, "f32", 2), (513, 33001, "f32", 2), (2600, 12001, "f16", 0)])
def test_gradients(size):
    import torch
    from cudeep_amd import ops
    rows, vocab, dtype, past = size
    assert _past(rows, vocab, dtype) == past
    say("past the caches", size)
    torch.manual_seed(0)
    x, t = _logits(rows, vocab, 1, dtype), _ints(0, vocab, (rows,), 2)
    idx, val, w = _ints(0, vocab, (rows, 12), 3), torch.randn(rows, 12, device="cuda"), torch.rand(rows, device="cuda")
    w[::5] = 0.0
    r = ops.token_logprobs(x, t, entropy=True)
    e = _check_logprobs(x, t, 1.0, r, 0)
    kw = dict(entropy=r.entropy, grad_entropy=w)
    dx = ops.token_logprobs_backward(w, x, t, r.stats, **kw)
    _check_backward(x, t, e, w, w, dx)
    del e
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    _check_distill(x, idx, val, 1.0, w, loss, grad)
    if dtype != "f32":   # what reads the gradient next sees all of it
        y, head = _logits(rows, 64, 4, dtype), _logits(vocab, 64, 5, dtype)
        want = ops.linear16_backward(grad.clone(), y, head, bias=False)
        for out in (None, x.clone()):
            again, g = ops.distill_loss(x if out is None else out, idx, val, weight=w, out=out)
            got = ops.linear16_backward(g, y, head, bias=False)
            assert torch.equal(again, loss) and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    same = x.clone()
    assert ops.distill_loss(same, idx, val, weight=w, out=same)[1] is same and torch.equal(same, grad)
    assert ops.token_logprobs_backward(w, x, t, r.stats, out=x, **kw) is x and torch.equal(x, dx)
