"""What reads a model's logits (token_logprobs, its backward pass, distill_loss) against the formulas in 64
bits.

Bounds.  Let d = (x - m) / T, with a difference rounded once, 1 / T once and their product once, and the
exponential's scaled argument twice more: an element's exp(d) is off by 5 2^-24 |d| and the hardware's
2^-22, and by 2^-22 for each time its sum is rescaled (at most once a round of 4096 elements or fewer, and
ten joins).  Weighted with p, |d| averages to less than ln V + 1.  So S is off by
5 U (ln V + 1) + 2^-22 (rounds + 11) + U (rounds + 50 additions), relative; L by that and two roundings of
L; l = d - L by three roundings of d and L's error.  The entropy L - sum p d takes S's error
on both and 5 U of sum p d^2.  A gradient's p is exp(l): l's error, relative, and the exponential's; results in 16
bits are off by half a step of their own."""
import math

import pytest

from tests.gpu_util import require_gpu, say

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _t():
    import torch
    return torch


def _ops():
    import cudeep_amd.ops as o
    return o


def _dtype(name):
    torch = _t()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def _logits(rows, vocab, seed, dtype, scale=3.0):
    torch = _t()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, vocab), device="cuda", generator=g) * scale).to(_dtype(dtype))


def _ints(lo, hi, shape, seed):
    torch = _t()
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, shape, device="cuda", generator=g)


def _sum_bound(vocab):
    rounds = -(-vocab // 4096) + 1
    return 5 * U * (math.log(vocab) + 1) + 2.0 ** -22 * (rounds + 11) + U * (rounds + 50)


class Exact:
    """The formulas in 64 bits, and how far a float32 result may be from them."""

    def __init__(self, x, T):
        torch = _t()
        x = x.double()
        self.T = T
        self.m = x.amax(-1, keepdim=True)
        self.d = (x - torch.where(self.m > -INF, self.m, 0.0)) / T
        self.L = torch.logsumexp(self.d, -1, keepdim=True)
        some = self.L > -INF
        self.l = torch.where(some, self.d - torch.where(some, self.L, 0.0), -INF)
        self.p = torch.exp(self.l)
        self.some = some
        zero = torch.zeros_like(self.p)
        self.H = -torch.where(self.p > 0, self.p * self.l, zero).sum(-1)
        sb = _sum_bound(x.shape[1])
        pd = torch.where(self.p > 0, self.p * self.d, zero)
        mean, square = pd.sum(-1).abs(), torch.where(self.p > 0, pd * self.d, zero).sum(-1)
        labs = torch.where(some, self.L, 0.0).abs()
        dabs = torch.where(self.d > -INF, self.d, zero).abs()   # (-infinity is exact)
        self.l_bound = 4 * U * (dabs + labs + torch.where(self.l > -INF, self.l, zero).abs()) + sb
        self.h_bound = sb * (2 + 2 * mean) + 8 * U * (square + mean + labs[:, 0] + 1)


def _near(got, want, bound, what):
    """got within bound of want and their own type's rounding; infinities and NaN the same."""
    torch = _t()
    g, w = got.double(), want.double()
    assert g.shape == w.shape, what
    # what lies past the type's largest value rounds to an infinity
    w = torch.where(w.abs() > torch.finfo(got.dtype).max, w.sign() * INF, w)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    far = torch.isinf(w) | torch.isinf(g)
    assert torch.equal(g[far], w[far]), what
    ok = torch.isfinite(w)
    if ok.any():
        bound = torch.as_tensor(bound, device=w.device, dtype=torch.float64).expand_as(w)[ok]
        rel = torch.finfo(got.dtype).eps / 2
        least = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126}[got.dtype]
        over = ((g[ok] - w[ok]).abs() - bound * (1 + rel) - rel * w[ok].abs() - least).max()
        assert float(over) <= 0, (what, float(over))


def _top(x, k):
    """The k largest of each row, the lowest index first among equals."""
    torch = _t()
    v, i = torch.sort(x.double() + 0.0, dim=1, descending=True, stable=True)
    return i[:, :k]


def _check_logprobs(x, t, T, r, top):
    torch = _t()
    e = Exact(x, T)
    at = t.clamp_min(0)[:, None]
    want = torch.where(t >= 0, e.l.gather(1, at)[:, 0], 0.0)
    _near(r.logprob, want, e.l_bound.gather(1, at)[:, 0], "logprob")
    if r.entropy is not None:
        _near(r.entropy, e.H, e.h_bound, "entropy")
    if top:
        i = _top(x, top)
        assert torch.equal(r.top_index, i)
        _near(r.top_logprob, e.l.gather(1, i), e.l_bound.gather(1, i), "top_logprob")
    return e


def _check_backward(x, t, e, g, gh, dx):
    torch = _t()
    at = t.clamp_min(0)[:, None]
    gg = torch.where(t >= 0, g.double(), 0.0)[:, None] if g is not None else torch.zeros_like(e.L)
    h = gh.double()[:, None] if gh is not None else torch.zeros_like(e.L)
    zero = torch.zeros_like(e.p)
    l = torch.where(e.p > 0, e.l, zero)
    H = e.H[:, None]
    want = (-gg * e.p - h * e.p * (l + H)) / e.T
    want = torch.where(e.some, want.scatter_add(1, at, gg / e.T), zero)
    size = e.p * (h.abs() * (l.abs() + H.abs()) + gg.abs())
    bound = (size * (e.l_bound + 2.0 ** -20) + e.p * h.abs() * (e.l_bound + e.h_bound[:, None])) / e.T
    bound = bound.scatter_add(1, at, 4 * U * gg.abs() / e.T)
    # an exponential below 2^-126 is 0
    _near(dx, want, bound + 2.0 ** -126 * (gg.abs() + h.abs() * 200) / e.T, "gradient")


SIZES = [(1, 1), (1, 2), (3, 7), (2, 64), (5, 255), (3, 257), (1, 4097), (1, 32000), (5, 50001), (300, 1000),
         (130, 8200), (33, 33000), (1030, 3001), (2, 200003), (1100, 8192), (1025, 5003)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", SIZES)
def test_logprobs(size, dtype):
    torch, ops = _t(), _ops()
    rows, vocab = size
    x, t = _logits(rows, vocab, 1, dtype), _ints(0, vocab, (rows,), 2)
    t[::5] = -100 if rows > 5 else t[::5]
    for T, top, entropy in ((1.0, 0, False), (0.7, min(5, vocab), True), (3.0, min(64, vocab), False), (1.0, 0, True)):
        say("token_logprobs", size, dtype, T, top, entropy)
        r = ops.token_logprobs(x, t, temperature=T, top=top, entropy=entropy)
        e = _check_logprobs(x, t, T, r, top)
        assert (r.entropy is None) == (not entropy) and (r.top_index is None) == (not top)
        g = torch.randn(rows, device="cuda")
        gh = torch.randn(rows, device="cuda") if entropy else None
        dx = ops.token_logprobs_backward(g, x, t, r.stats, entropy=r.entropy, grad_entropy=gh, temperature=T)
        _check_backward(x, t, e, g, gh, dx)
        if entropy:
            dx = ops.token_logprobs_backward(None, x, t, r.stats, entropy=r.entropy, grad_entropy=gh, temperature=T)
            _check_backward(x, t, e, None, gh, dx)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [2, 1100])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_alternatives_of_rows_in_an_order(top, rows, dtype):
    """Equal logits, rising, falling, and all large ones with a few threads: more candidates than the
    usual few."""
    torch, ops = _t(), _ops()
    vocab = 50003 if rows == 2 else 9001
    say("top", top, rows, dtype)
    n = torch.arange(vocab, device="cuda")
    kinds = [torch.zeros(vocab, device="cuda"), n / 100.0, -n / 100.0, (n // 8 % 256 < 3) * 50.0 + n % 7,
             (n // 4 % 256 < 2) * 50.0 - n / 1000.0, (n % 2) * 1.0, torch.where(n == vocab - 1, 9.0, -INF),
             torch.where(n % 1000 == 7, 1.0, -INF), torch.where(n % 3 == 0, -0.0, 0.0),
             torch.where(n % 2 == 0, -INF, torch.finfo(_dtype(dtype)).min), torch.full((vocab,), -INF, device="cuda")]
    x = torch.stack([kinds[r % len(kinds)] for r in range(max(rows, len(kinds)))]).to(_dtype(dtype))
    for part in ([x[i:i + rows] for i in range(0, len(x), rows)] if rows == 2 else [x]):
        r = ops.token_logprobs(part, torch.zeros(len(part), dtype=torch.int64, device="cuda"), top=top)
        assert torch.equal(r.top_index, _top(part, top))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(12, 40), (12, 9000), (1200, 700), (1200, 9000)])
def test_masks(size, dtype):
    """-infinity and the type's lowest value as masks: part of a row, all but one, all of it, the token's own."""
    torch, ops = _t(), _ops()
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
    x[9::12, : vocab - 2] = -INF
    for T in (1.0, 0.01, 100.0):
        say("masks", size, dtype, T)
        top = min(20, vocab)
        r = ops.token_logprobs(x, t, temperature=T, entropy=True, top=top)
        e = _check_logprobs(x, t, T, r, top)
        assert (r.logprob[2::12] == -INF).all() and (r.entropy[2::12] == 0).all()
        g, gh = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
        dx = ops.token_logprobs_backward(g, x, t, r.stats, entropy=r.entropy, grad_entropy=gh, temperature=T)
        assert (dx[2::12] == 0).all()
        _check_backward(x, t, e, g, gh, dx)


@pytest.mark.parametrize("rows", [9, 1200])
def test_nan_and_infinity_stay_in_their_rows(rows):
    torch, ops = _t(), _ops()
    x, t = _logits(rows, 9000, 5, "f32"), _ints(0, 9000, (rows,), 6)
    idx, val = _ints(0, 9000, (rows, 8), 7), torch.randn(rows, 8, device="cuda")
    w, g = torch.rand(rows, device="cuda"), torch.randn(rows, device="cuda")
    clean = ops.token_logprobs(x, t, entropy=True, top=5)
    closs, cgrad = ops.distill_loss(x, idx, val, weight=w)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[1, 3, 5]] = True
    x[1, 77], x[3, 8999], x[5] = float("nan"), INF, float("nan")
    r = ops.token_logprobs(x, t, entropy=True, top=5)
    for a, b in zip(r, clean):
        if a is not r.stats:
            assert torch.equal(a[~bad], b[~bad])
    assert torch.equal(r.stats[:, ~bad], clean.stats[:, ~bad])
    assert torch.isnan(r.logprob[bad]).all() and torch.isnan(r.entropy[bad]).all() and torch.isnan(r.top_logprob[bad]).all()
    assert ((r.top_index >= 0) & (r.top_index < 9000)).all()
    dx = ops.token_logprobs_backward(g, x, t, r.stats)
    assert torch.isnan(dx[bad]).all() and torch.isfinite(dx[~bad]).all()
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    assert torch.equal(loss[~bad], closs[~bad]) and torch.equal(grad[~bad], cgrad[~bad])
    assert torch.isnan(loss[bad]).all() and torch.isnan(grad[bad]).all()
    # rows that do not count stay out of it, whatever they hold
    g[bad], w[bad] = 0.0, 0.0
    assert (ops.token_logprobs_backward(g, x, t, r.stats)[bad] == 0).all()
    assert (ops.distill_loss(x, idx, val, weight=w)[1][bad] == 0).all()


def test_indices_past_the_vocabulary():
    torch, ops = _t(), _ops()
    for rows in (4, 1200):
        x, t = _logits(rows, 9000, 5, "bf16"), _ints(0, 9000, (rows,), 6)
        t[1], t[2] = 9000, 2 ** 40
        r = ops.token_logprobs(x, t, top=3)
        assert torch.isnan(r.logprob[1:3]).all() and torch.isfinite(r.logprob[3:]).all() and torch.isfinite(r.top_logprob).all()
        dx = ops.token_logprobs_backward(torch.ones(rows, device="cuda"), x, t, r.stats)
        assert torch.isnan(dx[1:3]).all() and torch.isfinite(dx[3:]).all()
        idx, val = _ints(0, 9000, (rows, 8), 7), torch.randn(rows, 8, device="cuda")
        idx[1, 3], idx[2, 0] = 9000, 2 ** 40
        loss, grad = ops.distill_loss(x, idx, val, weight=torch.ones(rows, device="cuda"))
        assert torch.isnan(loss[1:3]).all() and torch.isnan(grad[1:3]).all()
        assert torch.isfinite(loss[3:]).all() and torch.isfinite(grad[3:]).all()


def _check_distill(x, idx, val, T, w, loss, grad):
    torch = _t()
    e = Exact(x, T)
    there, at = idx >= 0, idx.clamp_min(0).long()
    v = torch.where(there, val.double() / T, -INF)
    top = v.amax(-1, keepdim=True) if v.shape[1] else torch.full((len(x), 1), -INF, device="cuda").double()
    counts = top > -INF
    dv = v - torch.where(counts, top, 0.0)
    z = torch.logsumexp(dv, -1, keepdim=True) if v.shape[1] else top
    lq = torch.where(counts & (dv > -INF), dv - torch.where(counts, z, 0.0), -INF)
    q = torch.exp(lq)
    zero = torch.zeros_like(q)
    lq0, l = torch.where(q > 0, lq, zero), e.l.gather(1, at)
    want = torch.where(q > 0, q * (lq0 - l), zero).sum(-1)
    # q: roundings of its exponent, exp's own few, its sum's
    rel = 8 * U * (torch.where(q > 0, dv, zero).abs() + lq0.abs() + 8) + (q.shape[1] + 8) * U
    size = torch.where(q > 0, lq0.abs() + torch.where(l > -INF, l, zero).abs(), zero)
    bound = (q * (rel * (size + 1) + (q.shape[1] + 4) * U * size + e.l_bound.gather(1, at))).sum(-1)
    _near(loss, want, bound, "loss")
    if grad is None:
        return
    f = w.double()[:, None] / T
    both = (e.p.scatter_add(1, at, -q)) * f
    both = torch.where(counts & e.some, both, torch.zeros_like(both))
    gb = e.p * f.abs() * (e.l_bound + 2.0 ** -20)
    gb = gb.scatter_add(1, at, q * f.abs() * (rel + (q.shape[1] + 4) * U))
    _near(grad, both, gb + 2.0 ** -126 * f.abs(), "gradient")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [(1, 1, 1), (1, 5, 3), (2, 300, 7), (1, 32000, 16), (16, 40001, 64), (300, 1000, 1),
                                  (33, 33000, 200), (700, 3001, 20), (2, 200003, 1024), (257, 16411, 64)])
def test_distill(size, dtype):
    torch, ops = _t(), _ops()
    rows, vocab, count = size
    x = _logits(rows, vocab, 1, dtype)
    for n, T in enumerate((1.0, 2.0, 0.5)):
        say("distill", size, dtype, T)
        idx, val = _ints(0, vocab, (rows, count), 2 + n), _logits(rows, count, 9 + n, ("f32", "bf16", "f16")[n])
        if n:   # lists of their own lengths, some of none
            keep = _ints(0, count + 1, (rows, 1), 3)
            idx = torch.where(torch.arange(count, device="cuda") < keep, idx, -1)
        if n == 2:
            idx, val = idx.to(torch.int32), torch.where(_ints(0, 3, (rows, count), 5) == 0, -INF, val)
        w = torch.rand(rows, device="cuda") - 0.3
        w[::7] = 0.0
        loss, grad = ops.distill_loss(x, idx, val, temperature=T, weight=w)
        _check_distill(x, idx, val, T, w, loss, grad)
        assert torch.equal(ops.distill_loss(x, idx, val, temperature=T), loss)


@pytest.mark.parametrize("rows", [3, 700])
def test_distill_entries_of_the_same_token(rows):
    torch, ops = _t(), _ops()
    x, w = _logits(rows, 9000, 1, "f32"), torch.rand(rows, device="cuda")
    idx, val = _ints(0, 5, (rows, 40), 2), torch.randn(rows, 40, device="cuda")
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    _check_distill(x, idx, val, 1.0, w, loss, grad)


@pytest.mark.parametrize("rows", [3, 700])
def test_distill_without_entries_and_masked_students(rows):
    torch, ops = _t(), _ops()
    x, w = _logits(rows, 9000, 1, "bf16"), torch.ones(rows, device="cuda")
    loss, grad = ops.distill_loss(x, torch.empty((rows, 0), dtype=torch.int64, device="cuda"),
                                  torch.empty((rows, 0), device="cuda"), weight=w)
    assert (loss == 0).all() and (grad == 0).all()
    idx, val = _ints(0, 9000, (rows, 8), 2), torch.randn(rows, 8, device="cuda")
    x[0] = -INF                       # nothing left
    x[1, idx[1, 3]] = -INF            # what the teacher wants is masked
    x[2, ::2] = torch.finfo(x.dtype).min
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    assert loss[0] == INF and loss[1] == INF and (grad[0] == 0).all() and torch.isfinite(grad).all()
    _check_distill(x[1:], idx[1:], val[1:], 1.0, w[1:], loss[1:], grad[1:])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(3, 9001), (1200, 1003), (700, 2050)])
def test_in_place_and_views(size, dtype):
    """Logits inside a larger matrix of NaN, at odd offsets, the gradient in their own place or in another
    matrix, which is left as it was around it."""
    torch, ops = _t(), _ops()
    rows, vocab = size
    x, t = _logits(rows, vocab, 1, dtype), _ints(0, vocab, (rows,), 2)
    idx, val, w = _ints(0, vocab, (rows, 9), 3), torch.randn(rows, 9, device="cuda"), torch.rand(rows, device="cuda")
    r = ops.token_logprobs(x, t, entropy=True, top=5)
    dx = ops.token_logprobs_backward(w, x, t, r.stats, entropy=r.entropy, grad_entropy=w)
    loss, grad = ops.distill_loss(x, idx, val, weight=w)
    for lead, tail in ((0, 8), (3, 2), (1, 0)):
        say("views", size, dtype, lead, tail)
        big = torch.full((rows + 2, vocab + lead + tail), float("nan"), dtype=x.dtype, device="cuda")
        v = big[1:-1, lead:lead + vocab]
        v.copy_(x)
        r2 = ops.token_logprobs(v, t, entropy=True, top=5)
        assert all(torch.equal(a, b) for a, b in zip(r2, r))
        wide = torch.full((rows, vocab + 5), 7.0, dtype=x.dtype, device="cuda")
        assert torch.equal(ops.token_logprobs_backward(w, v, t, r.stats, entropy=r.entropy, grad_entropy=w,
                                                       out=wide[:, 2:2 + vocab]), dx)
        assert (wide[:, :2] == 7).all() and (wide[:, 2 + vocab:] == 7).all()
        l2, g2 = ops.distill_loss(v, idx, val, weight=w, out=v)
        assert g2 is v and torch.equal(l2, loss) and torch.equal(v, grad)
        v.copy_(x)
        assert ops.token_logprobs_backward(w, v, t, r.stats, entropy=r.entropy, grad_entropy=w, out=v) is v
        assert torch.equal(v, dx)
        v.fill_(float("nan"))
        assert torch.isnan(big).all()


def test_leading_dimensions():
    torch, ops = _t(), _ops()
    x, t = _logits(12, 500, 1, "f16").view(3, 4, 500), _ints(0, 500, (3, 4), 2)
    r = ops.token_logprobs(x, t, top=4)
    assert r.logprob.shape == (12,) and r.top_index.shape == (12, 4)
    dx = ops.token_logprobs_backward(torch.ones(12, device="cuda"), x, t, r.stats)
    idx, val = _ints(0, 500, (3, 4, 6), 3), torch.randn(3, 4, 6, device="cuda")
    loss, grad = ops.distill_loss(x, idx, val, weight=torch.ones(3, 4, device="cuda"))
    assert dx.shape == grad.shape == x.shape and loss.shape == (12,)
    one = ops.token_logprobs(x[0, 0], t[0, :1], top=4)
    assert torch.equal(one.top_index[0], r.top_index[0])
    assert ops.token_logprobs(x[:0].reshape(0, 500), t[:0].reshape(0)).logprob.shape == (0,)
    assert ops.distill_loss(x[:0].reshape(0, 500), idx[:0].reshape(0, 6), val[:0].reshape(0, 6)).shape == (0,)


def test_large_magnitudes():
    """Logits of 1e4 and more: differences are formed before they are scaled."""
    torch, ops = _t(), _ops()
    for rows, vocab in ((4, 9000), (1200, 900)):
        x = _logits(rows, vocab, 1, "f32") + 20000.0 * torch.randn(rows, 1, device="cuda")
        t = _ints(0, vocab, (rows,), 2)
        r = ops.token_logprobs(x, t, entropy=True, temperature=0.5)
        e = _check_logprobs(x, t, 0.5, r, 0)
        g = torch.randn(rows, device="cuda")
        dx = ops.token_logprobs_backward(g, x, t, r.stats, entropy=r.entropy, grad_entropy=g, temperature=0.5)
        _check_backward(x, t, e, g, g, dx)


def test_gradients_against_differences():
    """Central differences of the forward passes in 64 bits' formula and of the kernels themselves: the loss
    of a float32 row changes by 2 h grad + O(h^3), measured against roundings of a few 2^-22."""
    torch, ops = _t(), _ops()
    x, t = _logits(3, 60, 1, "f32", 1.0), _ints(0, 60, (3,), 2)
    idx, val = _ints(0, 60, (3, 5), 3), torch.randn(3, 5, device="cuda")
    one = torch.ones(3, device="cuda")
    T, h = 1.5, 2.0 ** -5
    r = ops.token_logprobs(x, t, entropy=True, temperature=T)
    dl = ops.token_logprobs_backward(one, x, t, r.stats, temperature=T)
    dh = ops.token_logprobs_backward(None, x, t, r.stats, entropy=r.entropy, grad_entropy=one, temperature=T)
    _, dd = ops.distill_loss(x, idx, val, weight=one, temperature=T)
    # rows of single changes, all at once
    up = (x[:, None, :] + h * torch.eye(60, device="cuda")).view(-1, 60)
    down = (x[:, None, :] - h * torch.eye(60, device="cuda")).view(-1, 60)
    tt, ii, vv = t.repeat_interleave(60), idx.repeat_interleave(60, 0), val.repeat_interleave(60, 0)
    a = ops.token_logprobs(up, tt, entropy=True, temperature=T)
    b = ops.token_logprobs(down, tt, entropy=True, temperature=T)
    # third derivatives of log sum exp and of the entropy are below 1 and (ln 60 + 4) in units of T^-3;
    # h^2 / 6 of them, and two values of up to 8 rounded 20 times over 2 h
    err = h * h / 6 + 2 * 20 * 8 * U / (2 * h)
    near = lambda got, lo, hi, s: float((got - ((hi - lo) / (2 * h)).view(3, 60)).abs().max()) < s * err
    assert near(dl, b.logprob, a.logprob, 1.0)
    assert near(dh, b.entropy, a.entropy, 9.0)
    assert near(dd, ops.distill_loss(down, ii, vv, temperature=T), ops.distill_loss(up, ii, vv, temperature=T), 1.0)


@pytest.mark.parametrize("rows", [2, 300, 1100])
def test_the_same_bits_every_time_and_in_a_graph(rows):
    torch, ops = _t(), _ops()
    vocab = 40000 if rows == 2 else 9000
    say("logits graph", rows)
    x, t = _logits(rows, vocab, 1, "bf16"), _ints(0, vocab, (rows,), 2)
    idx, val, w = _ints(0, vocab, (rows, 9), 3), torch.randn(rows, 9, device="cuda"), torch.rand(rows, device="cuda")
    ws = torch.empty(max(ops.token_logprobs_workspace_bytes(rows, vocab, 5),
                         ops.distill_loss_workspace_bytes(rows, vocab, 9), 1), dtype=torch.uint8, device="cuda")

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
    for k in range(3):
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
    torch, ops = _t(), _ops()
    x, t = _logits(3, 60000, 1, "f32"), _ints(0, 60000, (3,), 2)
    idx, val, w = _ints(0, 60000, (3, 9), 3), torch.randn(3, 9, device="cuda"), torch.rand(3, device="cuda")

    def step():
        return tuple(ops.token_logprobs(x, t, entropy=True, top=5)) + ops.distill_loss(x, idx, val, weight=w)

    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(8):
        with torch.cuda.stream(streams[k % 2]):
            got.append(step())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_offsets_past_32_bits():
    """More than 2^32 bytes, and 2^31 elements, of logits: the last rows are those of a small batch."""
    torch, ops = _t(), _ops()
    rows, vocab = 34000, 65536
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device="cuda")
    x[-3:] = _logits(3, vocab, 1, "bf16")
    t = torch.zeros(rows, dtype=torch.int64, device="cuda")
    t[-3:] = _ints(0, vocab, (3,), 2)
    idx = torch.zeros((rows, 4), dtype=torch.int64, device="cuda")
    idx[-3:] = _ints(0, vocab, (3, 4), 3)
    val, w = torch.randn(rows, 4, device="cuda"), torch.ones(rows, device="cuda")
    r = ops.token_logprobs(x, t, entropy=True, top=3)
    e = _check_logprobs(x[-3:], t[-3:], 1.0, ops.TokenLogprobs(r.logprob[-3:], r.stats[:, -3:], *(a[-3:] for a in r[2:])), 3)
    dx = ops.token_logprobs_backward(w, x, t, r.stats, entropy=r.entropy, grad_entropy=w)
    _check_backward(x[-3:], t[-3:], e, w[-3:], w[-3:], dx[-3:])
    loss, grad = ops.distill_loss(x, idx, val, weight=w, out=dx)
    _check_distill(x[-3:], idx[-3:], val[-3:], 1.0, w[-3:], loss[-3:], grad[-3:])


def test_refusals():
    torch, ops = _t(), _ops()
    x, t = _logits(4, 100, 1, "f32"), _ints(0, 100, (4,), 2)
    idx, val, w = _ints(0, 100, (4, 5), 3), torch.randn(4, 5, device="cuda"), torch.rand(4, device="cuda")
    r = ops.token_logprobs(x, t)

    def refused(f, kind):
        with pytest.raises(kind):
            f()

    refused(lambda: ops.token_logprobs(x.double(), t), TypeError)
    refused(lambda: ops.token_logprobs(x.t(), t), ValueError)
    refused(lambda: ops.token_logprobs(x, t.int()), TypeError)
    refused(lambda: ops.token_logprobs(x, t[:3]), ValueError)
    refused(lambda: ops.token_logprobs(x, t.cpu()), ValueError)
    refused(lambda: ops.token_logprobs(x, t, top=65), RuntimeError)
    refused(lambda: ops.token_logprobs(x[:, :3], t, top=4), RuntimeError)
    refused(lambda: ops.token_logprobs(x[:, :0], t), RuntimeError)
    for T in (0.0, -1.0, float("nan"), float("inf"), 1e-7, 1e7):
        refused(lambda: ops.token_logprobs(x, t, temperature=T), RuntimeError)
        refused(lambda: ops.distill_loss(x, idx, val, temperature=T), RuntimeError)
    refused(lambda: ops.token_logprobs_backward(w, x, t, r.stats[:1]), ValueError)
    refused(lambda: ops.token_logprobs_backward(w, x, t, r.stats[:, :3]), ValueError)
    refused(lambda: ops.token_logprobs_backward(w.double(), x, t, r.stats), TypeError)
    refused(lambda: ops.token_logprobs_backward(w, x, t, r.stats, grad_entropy=w), ValueError)
    refused(lambda: ops.token_logprobs_backward(w, x, t, r.stats, out=x.half()), TypeError)
    refused(lambda: ops.token_logprobs_backward(w, x, t, r.stats, out=x[:3]), ValueError)
    big = _logits(5, 100, 1, "f32")
    refused(lambda: ops.token_logprobs_backward(w, big[:4], t, r.stats, out=big[1:]), RuntimeError)
    refused(lambda: ops.distill_loss(big[:4], idx, val, weight=w, out=big[1:]), RuntimeError)
    refused(lambda: ops.distill_loss(x, idx, val, out=x), ValueError)
    refused(lambda: ops.distill_loss(x, idx.float(), val), TypeError)
    refused(lambda: ops.distill_loss(x, idx, val.double()), TypeError)
    refused(lambda: ops.distill_loss(x, idx[:, :4], val), ValueError)
    refused(lambda: ops.distill_loss(x, idx[:3], val[:3]), ValueError)
    refused(lambda: ops.distill_loss(x, idx, val, weight=w[:3]), ValueError)
    many = torch.zeros((4, 1025), dtype=torch.int64, device="cuda")
    refused(lambda: ops.distill_loss(x, many, many.float()), RuntimeError)
