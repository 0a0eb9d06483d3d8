"""Results of what reads logits that lie over each other, or over what other workgroups of the call still read, are
refused before any launch (no GPU needed); gradients in the logits' own place, and neighbours, are not."""
import ctypes

import pytest

from cudeep_amd import _lib as L

F32, F16 = 0, 2
ROWS, VOCAB = 4, 70000


def _at(k, more=0):   # never dereferenced: the calls that are not refused are of 0 rows, or fail for their workspace
    return ctypes.c_void_p(0x100000 + 0x1000000 * k + more)


def _status(name, args):
    return getattr(L.lib(), name)(*args)


def _refused(name, good, at, value):
    args = list(good)
    args[at] = value
    assert _status(name, args) == L.CDX_ERR_INVALID_ARG, (name, at, value)
    said = L.lib().cdx_last_error()
    assert name.encode() in said and b"overlap" in said, said


# logits, ldx, rows, vocab, dtype, T, targets, logprob, stats, entropy, top, top_lp, top_index, ws, bytes, stream
LOGPROBS = [_at(0), VOCAB, ROWS, VOCAB, F32, 1.0, _at(1), _at(2), _at(3), _at(4), 5, _at(5), _at(6), _at(7), 16, None]
# g, logits, ldx, rows, vocab, dtype, T, targets, stats, entropy, gh, grad, ldg, stream
BACKWARD = [_at(0), _at(1), VOCAB, ROWS, VOCAB, F32, 1.0, _at(2), _at(3), _at(4), _at(5), _at(6), VOCAB, None]
# logits, ldx, rows, vocab, dtype, T, index, ldi, bytes, teacher, ldt, tdtype, count, loss, weight, grad, ldg, ws, n, s
DISTILL = [_at(0), VOCAB, ROWS, VOCAB, F32, 1.0, _at(1), 5, 8, _at(2), 5, F16, 5, _at(3), _at(4), _at(5), VOCAB, _at(7), 16,
           None]


def test_results_of_token_logprobs():
    for at, own in ((7, 2), (8, 3), (9, 4), (11, 5), (12, 6)):
        for k in range(7):
            if k != own:
                _refused("cdx_token_logprobs", LOGPROBS, at, _at(k))
    _refused("cdx_token_logprobs", LOGPROBS, 7, _at(0, 4 * ROWS * VOCAB - 4))   # the last logit
    _refused("cdx_token_logprobs", LOGPROBS, 7, _at(3, 4 * (2 * ROWS - 1)))     # the last of stats
    _refused("cdx_token_logprobs", LOGPROBS, 8, _at(1, 8 * ROWS - 4))           # the last target
    for value in (_at(0, 4 * ROWS * VOCAB), _at(3, 8 * ROWS), _at(1, 8 * ROWS)):
        args = list(LOGPROBS)
        args[7] = value
        assert _status("cdx_token_logprobs", args) == L.CDX_ERR_WORKSPACE   # refused for that alone


def test_gradients_of_log_probabilities():
    for k in (0, 2, 3, 4, 5):
        _refused("cdx_token_logprobs_backward", BACKWARD, 11, _at(k))
        # a vector inside the gradient's matrix
        _refused("cdx_token_logprobs_backward", BACKWARD, {0: 0, 2: 7, 3: 8, 4: 9, 5: 10}[k], _at(6, 4 * VOCAB + 64))


@pytest.mark.parametrize("grad", [_at(5), _at(0)])   # apart, and in the logits' place
def test_distillation(grad):
    good = list(DISTILL)
    good[15] = grad
    inside = ctypes.c_void_p(grad.value + 4 * VOCAB + 64)
    for at in (6, 9, 13, 14):
        _refused("cdx_distill_loss", good, at, inside)
    # the teacher's values as columns of the logits that the gradient replaces
    args = list(good)
    args[9], args[10], args[11] = grad, VOCAB, F32
    assert _status("cdx_distill_loss", args) == L.CDX_ERR_INVALID_ARG and b"teacher" in L.lib().cdx_last_error()
    for k in (0, 1, 2, 4):
        _refused("cdx_distill_loss", good, 13, _at(k))
    assert _status("cdx_distill_loss", good) == L.CDX_ERR_WORKSPACE
    # without a gradient nothing is written there
    args = list(good)
    args[9], args[10], args[11], args[14], args[15] = _at(0), VOCAB, F32, None, None
    assert _status("cdx_distill_loss", args) == L.CDX_ERR_WORKSPACE
