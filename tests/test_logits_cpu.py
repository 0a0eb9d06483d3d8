"""The C entry points of what reads logits refuse bad arguments before any launch, their size queries answer
without a GPU, and the wrappers refuse what is not on one."""
import ctypes

import pytest

from cudeep_amd import _lib as L

F32, F64, F16, BF16 = 0, 1, 2, 3


def _at(k):   # never dereferenced: validation fails first
    return ctypes.c_void_p(0x100000 + 0x1000000 * k)


def _status(name, *args):
    return getattr(L.lib(), name)(*args)


def _bad(name, good, changes):
    """Every change {position: value} of the good arguments is refused."""
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert _status(name, *args) == L.CDX_ERR_INVALID_ARG, (name, at, value)
        assert name.encode() in L.lib().cdx_last_error()


COMMON = [(2, -1), (2, 1 << 41), (3, 0), (3, 1 << 31), (4, F64), (4, 4), (5, 0.0), (5, -1.0), (5, float("nan")),
          (5, 1e7)]


def test_token_logprobs_arguments():
    # logits, ldx, rows, vocab, dtype, T, targets, logprob, stats, entropy, top, top_lp, top_index, ws, bytes, stream
    good = [_at(0), 100, 4, 100, F32, 1.0, _at(1), _at(2), _at(3), _at(4), 5, _at(5), _at(6), None, 0, None]
    _bad("cdx_token_logprobs", good, COMMON + [(0, None), (1, 99), (6, None), (7, None), (8, None), (10, -1), (10, 65),
                                               (11, None), (12, None)])
    few = list(good)
    few[3] = 4
    assert _status("cdx_token_logprobs", *few) == L.CDX_ERR_INVALID_ARG
    none = list(good)
    none[2] = 0
    assert _status("cdx_token_logprobs", *none) == L.CDX_OK
    small = list(good)
    small[1] = small[3] = 1 << 21
    small[13], small[14] = _at(7), 4
    assert _status("cdx_token_logprobs", *small) == L.CDX_ERR_WORKSPACE
    assert _status("cdx_token_logprobs_workspace_size", 1, 1 << 21, 5) > 0
    assert _status("cdx_token_logprobs_workspace_size", 8192, 100000, 5) == 0
    assert _status("cdx_token_logprobs_workspace_size", 1, 100000, 65) == 0


def test_backward_arguments():
    # g, logits, ldx, rows, vocab, dtype, T, targets, stats, entropy, gh, grad, ldg, stream
    good = [_at(0), _at(1), 100, 4, 100, F32, 1.0, _at(2), _at(3), _at(4), _at(5), _at(6), 100, None]
    _bad("cdx_token_logprobs_backward", good, [(at + 1, v) for at, v in COMMON] + [
        (1, None), (2, 99), (7, None), (8, None), (9, None), (11, None), (12, 99),
        (11, ctypes.c_void_p(_at(1).value + 4))])
    none = list(good)
    none[3] = 0
    assert _status("cdx_token_logprobs_backward", *none) == L.CDX_OK


def test_distill_arguments():
    # logits, ldx, rows, vocab, dtype, T, index, ldi, bytes, teacher, ldt, tdtype, count, loss, weight, grad, ldg, ws, n, s
    good = [_at(0), 100, 4, 100, F32, 1.0, _at(1), 5, 8, _at(2), 5, F32, 5, _at(3), _at(4), _at(5), 100, None, 0, None]
    _bad("cdx_distill_loss", good, COMMON + [
        (0, None), (1, 99), (6, None), (7, 4), (8, 2), (9, None), (10, 4), (11, F64), (12, -1), (12, 1025), (13, None),
        (15, None), (16, 99), (15, ctypes.c_void_p(_at(0).value + 4))])
    none = list(good)
    none[2] = 0
    assert _status("cdx_distill_loss", *none) == L.CDX_OK
    small = list(good)
    small[1] = small[3] = small[16] = 1 << 21
    small[17], small[18] = _at(7), 4
    assert _status("cdx_distill_loss", *small) == L.CDX_ERR_WORKSPACE
    assert _status("cdx_distill_loss_workspace_size", 8192, 100000, 5) == 0


def test_wrappers_refuse_host_tensors():
    torch = pytest.importorskip("torch")
    from cudeep_amd import ops
    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for f in (lambda: ops.token_logprobs(x, t), lambda: ops.token_logprobs_backward(x[:, 0], x, t, x[:, :2]),
              lambda: ops.distill_loss(x, t[:, None], x[:, :1])):
        with pytest.raises((ValueError, TypeError)):
            f()
