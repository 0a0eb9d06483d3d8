"""Long rows of logits that several workgroups share, joined by a second launch: each test asks the library that its
sizes are cut, so that it cannot come to test something else.  Bounds as in test_gpu_logits.py."""
import ctypes

import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_logits import (INF, _check_backward, _check_distill, _check_logprobs, _dtype, _ints, _logits, _top)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


@pytest.fixture(autouse=True)
def _seed(_gpu):
    _torch().manual_seed(0)


def _torch():
    import torch
    return torch


def _ops():
    from cudeep_amd import ops
    return ops


def _cut(rows, vocab, top=0, distill=True):
    """The parts that rows are cut into, by both operators."""
    from cudeep_amd import _lib as L
    f = L.lib().cdxi_logits_parts
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_int, ctypes.c_int64, ctypes.c_int64, ctypes.c_int]
    parts = f(0, rows, vocab, top)
    assert parts > 1 and _ops().token_logprobs_workspace_bytes(rows, vocab, top) > 0
    if distill:
        assert f(1, rows, vocab, 0) > 1 and _ops().distill_loss_workspace_bytes(rows, vocab, 1) > 0
    return parts


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("top", [1, 20, 64])
@pytest.mark.parametrize("vocab", [70001, 131077])
def test_alternatives_of_rows_in_an_order(vocab, top, dtype):
    """Equal logits in and across parts, rising, falling, large ones at the parts' ends, masks."""
    torch, ops = _torch(), _ops()
    n = torch.arange(vocab, device="cuda")
    low = torch.finfo(_dtype(dtype)).min
    kinds = [torch.zeros(vocab, device="cuda"), n / 5000.0, -n / 5000.0, (n // 8 % 256 < 3) * 50.0 + n % 7, (n % 2) * 1.0,
             torch.where(n == vocab - 1, 9.0, -INF), torch.where(n % 1000 == 7, 1.0, -INF), torch.where(n % 3 == 0, -0.0, 0.0),
             torch.where(n % 2 == 0, -INF, low), torch.full((vocab,), -INF, device="cuda"), torch.full((vocab,), low, device="cuda"),
             torch.where(n >= vocab - 3, 1.0, 0.0), torch.where(n % 64 == 0, 2.0, 1.0), torch.where(n < vocab // 2, -INF, 0.5),
             torch.where(n % 17536 >= 17534, 3.0, n / 1e6)]
    x = torch.stack(kinds).to(_dtype(dtype))
    for rows in (1, 2, len(kinds)):
        say("top in parts", vocab, top, dtype, rows, _cut(rows, vocab, top))
        for i in range(0, len(kinds), rows):
            part = x[i:i + rows]
            r = ops.token_logprobs(part, torch.zeros(len(part), dtype=torch.int64, device="cuda"), top=top)
            assert torch.equal(r.top_index, _top(part, top))


@pytest.mark.parametrize("vocab", [4210689, 4210690, 4210691])   # 257 parts, the last of 1 to 3 elements
@pytest.mark.parametrize("where", ["last", "equal", "masked"])
def test_a_last_part_of_few_elements(where, vocab):
    torch, ops = _torch(), _ops()
    assert _cut(1, vocab, 1) == 257
    say("last part", where, vocab)
    x, t = _logits(1, vocab, 1, "f32"), torch.full((1,), vocab - 1, device="cuda")
    if where == "last":
        x[0, -1] = 50.0
    elif where == "equal":
        x.fill_(1.5)
    else:
        x[0, -3:] = -INF
    r = ops.token_logprobs(x, t, entropy=True, top=1)
    e = _check_logprobs(x, t, 1.0, r, 1)
    g = torch.ones(1, device="cuda")
    dx = ops.token_logprobs_backward(g, x, t, r.stats, entropy=r.entropy, grad_entropy=g)
    _check_backward(x, t, e, g, g, dx)
    idx = torch.tensor([[vocab - 1, 0, vocab - 2, 5]], device="cuda")
    val = torch.randn(1, 4, device="cuda")
    loss, grad = ops.distill_loss(x, idx, val, weight=g)
    _check_distill(x, idx, val, 1.0, g, loss, grad)


def _in_float32(x, idx, val, T):
    """What a float32 computation at the ends of its range is given, for the formula in 64 bits.  A difference (x - m) / T
    past the type's largest value is an infinity, as of a masked logit.  A q below 2^-150, half of the least value,
    is 0, as of an entry that does not count (where its logit is masked too the formula's q times infinity is
    infinite, and 0 here)."""
    torch = _torch()
    xd = x.double()
    m = xd.amax(-1, keepdim=True)
    d = (xd - torch.where(m > -INF, m, 0.0)) / T
    q = torch.softmax(torch.where(idx >= 0, val.double() / T, -INF), -1)
    return torch.where(d < -torch.finfo(torch.float32).max, -INF, xd).to(x.dtype), torch.where(q < 2.0 ** -150, -1, idx)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(12, 70001), (60, 131077)])
def test_masks(size, dtype):
    torch, ops = _torch(), _ops()
    rows, vocab = size
    low = torch.finfo(_dtype(dtype)).min
    x, t = _logits(rows, vocab, 3, dtype), _ints(0, vocab, (rows,), 4)
    x[0::12, ::2] = -INF
    x[1::12, ::2] = low
    x[2::12] = -INF
    x[3::12] = low
    x[4::12, 1:] = -INF
    x[5::12, :-1] = low
    x[6::12, :vocab // 2] = low
    x[6::12, vocab // 2:] = -INF
    x[7::12] = -INF
    x[7::12, vocab - 1] = 2.0
    t[7::12] = vocab - 1
    t[8::12] = 0
    x[8::12, 0] = -INF
    x[9::12, :vocab - 2] = -INF
    x[10::12, 20000:60000] = -INF     # whole parts
    t[11::12] = -1
    idx, val, w = _ints(0, vocab, (rows, 8), 7), torch.randn(rows, 8, device="cuda"), torch.rand(rows, device="cuda")
    for T in (1.0, 0.01, 100.0):
        say("masks in parts", size, dtype, T, _cut(rows, vocab, 20))
        r = ops.token_logprobs(x, t, temperature=T, entropy=True, top=20)
        e = _check_logprobs(x, t, T, r, 20)
        assert (r.logprob[2::12] == -INF).all() and (r.entropy[2::12] == 0).all()
        g, gh = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
        dx = ops.token_logprobs_backward(g, x, t, r.stats, entropy=r.entropy, grad_entropy=gh, temperature=T)
        assert (dx[2::12] == 0).all()
        _check_backward(x, t, e, g, gh, dx)
        some = torch.ones(rows, dtype=torch.bool, device="cuda")
        some[2::12] = False
        loss, grad = ops.distill_loss(x, idx, val, temperature=T, weight=w)
        assert (loss[2::12] == INF).all() and (grad[2::12] == 0).all()
        if dtype == "f32" and T == 1.0:
            # Rows 5: every entry is at l = -M, M the largest float32.  The loss is M times the sum of the q, which is 1
            # to within (8 + count) roundings of 2^-24, as M is M to within half a step; from M (1 + 2^-25) on a float32
            # is infinite.  So both M, less 2^-19 of it, and infinity are roundings of the exact loss.
            assert (loss[5::12] >= torch.finfo(torch.float32).max * (1 - 2.0 ** -19)).all()
            some[5::12] = False
        xs, ids = _in_float32(x[some], idx[some], val[some], T)
        _check_distill(xs, ids, val[some], T, w[some], loss[some], grad[some])


def test_nan_and_infinity_stay_in_their_rows():
    torch, ops = _torch(), _ops()
    rows, vocab = 9, 70001
    say("nan in parts", _cut(rows, vocab, 5))
    x, t = _logits(rows, vocab, 5, "f32"), _ints(0, vocab, (rows,), 6)
    idx, val = _ints(0, vocab, (rows, 8), 7), torch.randn(rows, 8, device="cuda")
    w, g = torch.rand(rows, device="cuda"), torch.randn(rows, device="cuda")
    clean = ops.token_logprobs(x, t, entropy=True, top=5)
    closs, cgrad = ops.distill_loss(x, idx, val, weight=w)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[1, 3, 5, 7]] = True
    x[1, 77], x[3, vocab - 1], x[5], x[7, 40000] = float("nan"), INF, float("nan"), float("nan")
    r = ops.token_logprobs(x, t, entropy=True, top=5)
    for a, b in zip(r, clean):
        if a is not r.stats:
            assert torch.equal(a[~bad], b[~bad])
    assert torch.equal(r.stats[:, ~bad], clean.stats[:, ~bad])
    assert torch.isnan(r.logprob[bad]).all() and torch.isnan(r.entropy[bad]).all() and torch.isnan(r.top_logprob[bad]).all()
    assert ((r.top_index >= 0) & (r.top_index < vocab)).all()
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    assert torch.equal(loss[~bad], closs[~bad]) and torch.equal(grad[~bad], cgrad[~bad])
    assert torch.isnan(loss[bad]).all() and torch.isnan(grad[bad]).all()
    w[bad] = 0.0
    assert (ops.distill_loss(x, idx, val, weight=w)[1][bad] == 0).all()


def test_indices_past_the_vocabulary():
    torch, ops = _torch(), _ops()
    rows, vocab = 4, 70001
    say("indices in parts", _cut(rows, vocab, 3))
    x, t = _logits(rows, vocab, 5, "bf16"), _ints(0, vocab, (rows,), 6)
    t[1], t[2] = vocab, 2 ** 40
    r = ops.token_logprobs(x, t, top=3)
    assert torch.isnan(r.logprob[1:3]).all() and torch.isfinite(r.logprob[[0, 3]]).all() and torch.isfinite(r.top_logprob).all()
    idx, val = _ints(0, vocab, (rows, 8), 7), torch.randn(rows, 8, device="cuda")
    idx[1, 3], idx[2, 0], idx[3, 5] = vocab, 2 ** 40, -7
    w = torch.ones(rows, device="cuda")
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    assert torch.isnan(loss[1:3]).all() and torch.isnan(grad[1:3]).all()
    good = torch.tensor([0, 3], device="cuda")
    _check_distill(x[good], idx[good], val[good], 1.0, w[good], loss[good], grad[good])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(1, 65536, 1), (2, 70001, 40), (33, 131077, 1024), (127, 70001, 64), (3, 200003, 1023)])
def test_distill(size, dtype):
    torch, ops = _torch(), _ops()
    rows, vocab, count = size
    x = _logits(rows, vocab, 1, dtype)
    for n, T in enumerate((1.0, 2.0, 0.5)):
        say("distill in parts", size, dtype, T, _cut(rows, max(vocab, 65537)))
        # every token many times, with ends of parts among them; then anywhere
        idx = (_ints(0, 5, (rows, count), 2) * 17536 - _ints(0, 2, (rows, count), 3)).clamp(0, vocab - 1) if n == 0 else \
            _ints(0, vocab, (rows, count), 2 + n)
        val = _logits(rows, count, 9 + n, ("f32", "bf16", "f16")[n])
        if n:
            keep = _ints(0, count + 1, (rows, 1), 3)
            idx = torch.where(torch.arange(count, device="cuda") < keep, idx, -1)
        if n == 2:
            idx, val = idx.to(torch.int32), torch.where(_ints(0, 3, (rows, count), 5) == 0, -INF, val)
        w = torch.rand(rows, device="cuda") - 0.3
        w[::7] = 0.0
        loss, grad = ops.distill_loss(x, idx, val, temperature=T, weight=w)
        _check_distill(x, idx, val, T, w, loss, grad)
        assert torch.equal(ops.distill_loss(x, idx, val, temperature=T), loss)
        again, same = ops.distill_loss(x.clone(), idx, val, temperature=T, weight=w)
        assert torch.equal(again, loss) and torch.equal(same, grad)


def test_distill_without_entries_and_masked_students():
    torch, ops = _torch(), _ops()
    rows, vocab = 3, 70001
    say("distill without entries", _cut(rows, vocab))
    x, w = _logits(rows, vocab, 1, "bf16"), torch.ones(rows, device="cuda")
    loss, grad = ops.distill_loss(x, torch.empty((rows, 0), dtype=torch.int64, device="cuda"),
                                  torch.empty((rows, 0), device="cuda"), weight=w)
    assert (loss == 0).all() and (grad == 0).all()
    idx, val = _ints(0, vocab, (rows, 8), 2), torch.randn(rows, 8, device="cuda")
    x[0] = -INF                       # nothing left
    x[1, idx[1, 3]] = -INF            # what the teacher wants is masked
    x[2, ::2] = torch.finfo(x.dtype).min
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    assert loss[0] == INF and loss[1] == INF and (grad[0] == 0).all() and torch.isfinite(grad).all()
    _check_distill(x[1:], idx[1:], val[1:], 1.0, w[1:], loss[1:], grad[1:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(3, 70001), (40, 131077)])
def test_in_place_and_views(size, dtype):
    torch, ops = _torch(), _ops()
    rows, vocab = size
    x, t = _logits(rows, vocab, 1, dtype), _ints(0, vocab, (rows,), 2)
    idx, val, w = _ints(0, vocab, (rows, 9), 3), torch.randn(rows, 9, device="cuda"), torch.rand(rows, device="cuda")
    r = ops.token_logprobs(x, t, entropy=True, top=5)
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    _check_distill(x, idx, val, 1.0, w, loss, grad)
    for lead, tail in ((0, 8), (3, 2), (1, 0)):
        say("views in parts", size, dtype, lead, tail, _cut(rows, vocab, 5))
        big = torch.full((rows + 2, vocab + lead + tail), float("nan"), dtype=x.dtype, device="cuda")
        v = big[1:-1, lead:lead + vocab]
        v.copy_(x)
        assert all(torch.equal(a, b) for a, b in zip(ops.token_logprobs(v, t, entropy=True, top=5), r))
        wide = torch.full((rows, vocab + 5), 7.0, dtype=x.dtype, device="cuda")
        l2, g2 = ops.distill_loss(v, idx, val, weight=w, out=wide[:, 2:2 + vocab])
        assert torch.equal(l2, loss) and torch.equal(g2, grad)
        assert (wide[:, :2] == 7).all() and (wide[:, 2 + vocab:] == 7).all()
        l2, g2 = ops.distill_loss(v, idx, val, weight=w, out=v)
        assert g2 is v and torch.equal(l2, loss) and torch.equal(v, grad)
        v.fill_(float("nan"))
        assert torch.isnan(big).all()


@pytest.mark.parametrize("rows", [1, 2, 33])
def test_the_same_bits_every_time_and_in_a_graph(rows):
    torch, ops = _torch(), _ops()
    vocab = 131077
    say("graph of parts", rows, _cut(rows, vocab, 5))
    x, t = _logits(rows, vocab, 1, "bf16"), _ints(0, vocab, (rows,), 2)
    idx, val, w = _ints(0, vocab, (rows, 9), 3), torch.randn(rows, 9, device="cuda"), torch.rand(rows, device="cuda")
    ws = torch.empty(max(ops.token_logprobs_workspace_bytes(rows, vocab, 5), ops.distill_loss_workspace_bytes(rows, vocab, 9)),
                     dtype=torch.uint8, device="cuda")

    def step():
        r = ops.token_logprobs(x, t, entropy=True, top=5, workspace=ws)
        dx = ops.token_logprobs_backward(w, x, t, r.stats, entropy=r.entropy, grad_entropy=w)
        return tuple(r) + (dx,) + ops.distill_loss(x, idx, val, weight=w, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x.copy_(_logits(rows, vocab, 10 + k, "bf16"))
        want = step()
        torch.cuda.synchronize()
        for h in held:
            h.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_two_streams():
    """Calls in flight together, each with its own scratch and on other logits: shared partial sums would show."""
    torch, ops = _torch(), _ops()
    rows, vocab = 3, 131077
    say("streams of parts", _cut(rows, vocab, 5))
    sets = [(_logits(rows, vocab, 1 + k, "f32"), _ints(0, vocab, (rows,), 2 + k), _ints(0, vocab, (rows, 9), 3 + k),
             _logits(rows, 9, 4 + k, "f32"), torch.rand(rows, device="cuda")) for k in (0, 10)]

    def step(x, t, idx, val, w):
        return tuple(ops.token_logprobs(x, t, entropy=True, top=5)) + ops.distill_loss(x, idx, val, weight=w)

    want = [step(*s) for s in sets]
    assert not torch.equal(want[0][0], want[1][0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(16):
        with torch.cuda.stream(streams[k % 2]):
            got.append(step(*sets[k % 2]))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[k % 2]))
