"""Products of the 16-bit Linear layer that are summed in slices, and the slopes' column sums in parts, captured into
graphs and on two streams at once with different inputs.  Each test asks the library that its products are sliced."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.routes16 import linear16_kernel
from tests.test_gpu_linear16 import _act_code, _check_backward, _check_forward, _rnd

pytestmark = pytest.mark.gpu

# M, N, K of a layer, and its products in slices: forward, input gradient, weight gradient (aligned, unaligned, few
# and many rows)
LAYERS = [((64, 8192, 4096), "fi"), ((8192, 256, 784), "w"), ((16, 640, 6575), "f"), ((1777, 299, 203), "w"),
          ((136, 4136, 264), "i"), ((299, 203, 1777), "f")]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _sliced(size, which):
    """The library takes those products, and no others, in slices."""
    M, N, K = size
    # (dz lies in rows of whole 8 in the workspace)
    got = ""
    for kind, product, aligned in (("forward", (M, N, K), K % 8 == 0), ("input", (M, K, N), K % 8 == 0),
                                   ("weight", (N, K, M), N % 8 == 0 and K % 8 == 0)):
        if linear16_kernel(kind, *product, aligned)[1] > 1:
            got += kind[0]
    assert got == which, got


def _inputs(size, seed):
    M, N, K = size
    return (_rnd((M, K), seed, "bf16"), _rnd((N, K), seed + 1, "bf16", K ** -0.5), _rnd((N,), seed + 2, "bf16"),
            _rnd((M, N), seed + 3, "bf16"), _rnd((M, N), seed + 4, "bf16"))


def _step(x, w, b, res, dy, act, **kw):
    from cudeep_amd import ops
    y, z = ops.linear16(x, w, b, epilogue=act, residual=res, keep=True, **kw)
    return (y, z) + ops.linear16_backward(dy, x, w, z, epilogue=act, **kw)


@pytest.mark.parametrize("layer", LAYERS)
def test_in_a_graph(layer):
    import torch
    from cudeep_amd import ops
    size, which = layer
    _sliced(size, which)
    say("graph of slices", size)
    act = _act_code("gelu")
    inputs = _inputs(size, 1)
    ws = torch.empty(max(ops.linear16_workspace_bytes(*size), ops.linear16_backward_workspace_bytes(*size, act)),
                     dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*inputs, act, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _step(*inputs, act, workspace=ws)
    for k in range(4):
        for t, new in zip(inputs, _inputs(size, 10 + 10 * k)):
            t.copy_(new)
        want = _step(*inputs, act, workspace=ws)
        torch.cuda.synchronize()
        for t in held:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
        assert all(torch.equal(a, b) for a, b in zip(_step(*inputs, act), want))
    x, w, b, res, dy = inputs
    y, z, dx, dw, db = want
    _check_forward(x, w, b, "gelu", res, y, z)
    _check_backward(dy, x, w, z, "gelu", dx, dw, db)


@pytest.mark.parametrize("layer", LAYERS)
def test_two_streams(layer):
    """Calls in flight together on other inputs, each with scratch of its own: partial sums or a dz that they shared
    would show."""
    import torch
    size, which = layer
    _sliced(size, which)
    say("streams of slices", size)
    act = _act_code("silu")
    sets = [_inputs(size, seed) for seed in (1, 51)]
    want = [_step(*s, act) for s in sets]
    assert not any(torch.equal(a, b) for a, b in zip(*want))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for k in range(12):
        with torch.cuda.stream(streams[k % 2]):
            got.append(_step(*sets[k % 2], act))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[k % 2])), k
