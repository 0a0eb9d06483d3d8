"""Each kernel of a 16-bit Linear layer in each of its three products, at sizes that end inside tiles and steps,
with operands inside larger matrices of NaN; slices; results beside their inputs; offsets past 32 bits.
Bounds as in test_gpu_linear16.py."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.routes16 import linear16_kernel
from tests.test_gpu_linear16 import _act_code, _check_backward, _check_forward, _inside, _rnd

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _ops():
    import cudeep_amd.ops as o
    return o


def _torch():
    import torch
    return torch


def _padded(t, aligned, value=float("nan")):
    """A view of t's values whose rows begin at multiples of 16 bytes, or do not."""
    lead = 8 if aligned else 3
    return _inside(t, lead, 8 + -t.shape[1] % 8 if aligned else 8 + (t.shape[1] + 1) % 2, value)[1]


# (kernel, whether slices are added, aligned, a product's M, N, K); K is no multiple of 64
CASES = [("direct", False, True, 5, 304, 1000), ("direct", False, True, 30, 4040, 1096),
         ("direct", False, True, 128, 520, 72), ("direct", False, False, 60, 4001, 333),
         ("direct", False, False, 17, 3999, 65), ("ring 64", False, True, 296, 1000, 200),
         ("tall", False, True, 1304, 1288, 200), ("tall", False, True, 8200, 136, 4104),
         ("ring 64", True, True, 136, 264, 4136), ("ring 128", False, True, 1400, 1608, 264),
         ("ring 128", True, True, 264, 520, 90120), ("tile 128", False, True, 2104, 2184, 200),
         ("turns", False, True, 3600, 3592, 200), ("turns", True, True, 1000, 1104, 53352),
         ("tile 128", False, True, 72, 33000, 136), ("tile 128", False, True, 33000, 128, 136),
         ("any", False, False, 839, 953, 77), ("any", False, False, 50, 30001, 77), ("any", True, False, 299, 203, 1777),
         ("any 128", False, False, 1801, 1807, 93), ("any 128", True, False, 1336, 1441, 4106)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", CASES)
def test_forward(case, dtype):
    name, slices, aligned, M, N, K = case
    got = linear16_kernel("forward", M, N, K, aligned)
    assert got[0] == name and (got[1] > 1) == slices
    say("forward", case, dtype)
    x, w, b, res = (_rnd((M, K), 1, dtype), _rnd((N, K), 2, dtype, K ** -0.5), _rnd((N,), 3, "f32"), _rnd((M, N), 4, dtype))
    out = _padded(_torch().zeros_like(res), aligned, 7.0)
    y, z = _ops().linear16(_padded(x, aligned), _padded(w, aligned), b, epilogue=_act_code("gelu"),
                           residual=_padded(res, aligned), keep=True, out=out)
    assert y is out
    _check_forward(x, w, b, "gelu", res, y, z)
    y = _ops().linear16(_padded(x, aligned), _padded(w, aligned))
    _check_forward(x, w, None, "none", None, y)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", [c for c in CASES if c[0] != "direct"])
def test_input_gradient(case, dtype):
    name, slices, aligned, M, N, K = case
    got = linear16_kernel("input", M, N, K, aligned)
    assert got[0] == name and (got[1] > 1) == slices
    say("input", case, dtype)
    w, dy, x = _rnd((K, N), 2, dtype, K ** -0.5), _rnd((M, K), 1, dtype), _rnd((1, N), 1, dtype).expand(M, N)
    dx, dw, db = _ops().linear16_backward(_padded(dy, aligned), x.contiguous(), _padded(w, aligned), params=False)
    assert dw is None and db is None
    _check_backward(dy, x, w, None, "none", dx, None, None)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("case", [c for c in CASES if c[0] != "direct"])
def test_weight_gradient(case, dtype):
    torch = _torch()
    name, slices, aligned, M, N, K = case
    got = linear16_kernel("weight", M, N, K, aligned)
    assert got[0] == name and (got[1] > 1) == slices
    say("weight", case, dtype)
    x, dy, w = _rnd((K, N), 1, dtype), _rnd((K, M), 2, dtype), torch.zeros((M, N), dtype=torch.float32, device="cuda")
    w = w.to(x.dtype)
    for pd in (None, torch.float32):
        dx, dw, db = _ops().linear16_backward(_padded(dy, aligned), _padded(x, aligned), w, input=False, param_dtype=pd)
        assert dx is None and dw.dtype == db.dtype == (pd or x.dtype)
        _check_backward(dy, x, w, None, "none", None, dw, db)


@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_slopes_of_a_large_layer(act):
    """grad and z of more than 64 MB each (they pass the caches by), with a last piece of fewer than eight."""
    M, N, K = 8203, 4005, 64
    say("large slopes", act)
    x, w, dy, z = _rnd((M, K), 1, "bf16"), _rnd((N, K), 2, "bf16"), _rnd((M, N), 3, "bf16"), _rnd((M, N), 4, "bf16")
    dx, dw, db = _ops().linear16_backward(_padded(dy, True), x, w, _padded(z, False), epilogue=_act_code(act))
    _check_backward(dy, x, w, z, act, dx, dw, db)


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("first", [True, False])
def test_columns_beside_each_other(rows, first):
    torch, ops = _torch(), _ops()
    x, w = _rnd((rows, 64), 1, "bf16"), _rnd((64, 64), 2, "bf16")
    buf = torch.zeros(rows, 128, device="cuda", dtype=torch.bfloat16)
    a, b = (buf[:, :64], buf[:, 64:]) if first else (buf[:, 64:], buf[:, :64])
    say("linear16 beside", rows, first)
    want = ops.linear16(x, w)
    a.copy_(x)
    assert torch.equal(ops.linear16(a, w, out=b), want) and torch.equal(a, x)
    r = ops.token_logprobs(a, torch.zeros(rows, dtype=torch.int64, device="cuda"))
    g, t = torch.ones(rows, device="cuda"), torch.zeros(rows, dtype=torch.int64, device="cuda")
    want = ops.token_logprobs_backward(g, x, t, r.stats)
    assert torch.equal(ops.token_logprobs_backward(g, a, t, r.stats, out=b), want) and torch.equal(a, x)
    idx, val = torch.full((rows, 2), 3, device="cuda"), torch.zeros(rows, 2, device="cuda")
    want = ops.distill_loss(x, idx, val, weight=g)[1]
    assert torch.equal(ops.distill_loss(a, idx, val, weight=g, out=b)[1], want) and torch.equal(a, x)


@pytest.mark.parametrize("size", [(64, 2056), (2056, 64), (61, 2051)])
def test_offsets_past_32_bits(size):
    """More than 2^31 elements of x, or of z and the outputs: the last rows are those of a small batch."""
    torch, ops = _torch(), _ops()
    N, K = size
    M, some = 1050000, 40
    say("linear16 past 32 bits", size)
    w, b = _rnd((N, K), 1, "bf16", K ** -0.5), _rnd((N,), 2, "f32")
    xs, ds = _rnd((some, K), 3, "bf16"), _rnd((some, N), 4, "bf16")
    x, dy = (torch.zeros((M, n), dtype=torch.bfloat16, device="cuda") for n in (K, N))
    x[-some:], dy[-some:] = xs, ds
    y, z = ops.linear16(x, w, b, epilogue=_act_code("silu"), keep=True)
    _check_forward(xs, w, b, "silu", None, y[-some:], z[-some:])
    assert torch.equal(y[M // 2], y[0]) and torch.equal(y[-some - 1], y[0])
    del y
    dx, dw, db = ops.linear16_backward(dy, x, w, z, epilogue=_act_code("silu"))
    # (zeros add nothing, and round nothing)
    _check_backward(ds, xs, w, z[-some:], "silu", dx[-some:], dw, db)
    assert not dx[0].any() and not dx[M // 2].any() and not dx[-some - 1].any()
