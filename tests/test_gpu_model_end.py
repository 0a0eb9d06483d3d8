"""A model's last layers in 16 bits as they are used together: a residual block of two layers, the head over
an odd vocabulary with rows padded to whole pieces, both losses, and every gradient back to the block's input;
each step against 64 bits at the step's own inputs, the whole in a graph, and the log probabilities that a
decoder reads, token by token."""
import pytest

from tests.gpu_util import require_gpu, say
from tests.test_gpu_linear16 import _act_code, _check_backward, _check_forward, _rnd
from tests.test_gpu_logits import _check_distill, _check_logprobs, _ints
from tests.test_gpu_logits import _check_backward as _check_logprob_gradient

pytestmark = pytest.mark.gpu

D, H, V = 264, 1032, 5003


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    require_gpu()


def _model(dtype):
    import torch
    p = dict(w1=_rnd((H, D), 1, dtype, D ** -0.5), b1=_rnd((H,), 2, "f32"), w2=_rnd((D, H), 3, dtype, H ** -0.5),
             b2=_rnd((D,), 4, dtype), head=_rnd((V, D), 5, dtype, 3 * D ** -0.5))
    return p


def _logits_view(rows, dtype):
    """Rows padded to whole 16-byte pieces, NaN behind the vocabulary."""
    import torch
    return torch.full((rows, (V + 7) // 8 * 8), float("nan"), dtype=dtype, device="cuda")[:, :V]


def _run(p, s):
    """One step over s's tokens: every intermediate value and gradient, by name."""
    from cudeep_amd import ops
    gelu = _act_code("gelu")
    v = {}
    v["h"], v["z"] = ops.linear16(s["x"], p["w1"], p["b1"], epilogue=gelu, keep=True)
    v["y"] = ops.linear16(v["h"], p["w2"], p["b2"], residual=s["x"])
    v["logits"] = ops.linear16(v["y"], p["head"], out=_logits_view(len(s["x"]), s["x"].dtype))
    v["r"] = ops.token_logprobs(v["logits"], s["t"], entropy=True, top=4)
    v["loss"], v["g1"] = ops.distill_loss(v["logits"], s["idx"], s["val"], temperature=2.0, weight=s["w"],
                                          out=_logits_view(len(s["x"]), s["x"].dtype))
    v["g2"] = ops.token_logprobs_backward(s["g"], v["logits"], s["t"], v["r"].stats, entropy=v["r"].entropy,
                                          grad_entropy=s["w"], out=_logits_view(len(s["x"]), s["x"].dtype))
    v["dl"] = _logits_view(len(s["x"]), s["x"].dtype)
    v["dl"].copy_(v["g1"] + v["g2"])
    v["dy"], v["dhead"], _ = ops.linear16_backward(v["dl"], v["y"], p["head"], bias=False)
    v["dh"], v["dw2"], v["db2"] = ops.linear16_backward(v["dy"], v["h"], p["w2"])
    v["dx"], v["dw1"], v["db1"] = ops.linear16_backward(v["dh"], s["x"], p["w1"], v["z"], epilogue=gelu)
    v["dx"] += v["dy"]   # past the block
    return v


def _tokens(rows, dtype, seed):
    import torch
    s = dict(x=_rnd((rows, D), seed, dtype), t=_ints(0, V, (rows,), seed + 1), idx=_ints(0, V, (rows, 12), seed + 2),
             val=_rnd((rows, 12), seed + 3, "f32"), w=torch.full((rows,), 1.0 / rows, device="cuda"),
             g=_rnd((rows,), seed + 4, "f32", 1.0 / rows))
    s["t"][::6] = -100      # padding: no token, no teacher, no weight
    s["idx"][::6], s["w"][::6], s["g"][::6] = -1, 0.0, 0.0
    return s


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 7, 130, 1111])
def test_a_training_step(rows, dtype):
    import torch
    p, s = _model(dtype), _tokens(rows, dtype, 10)
    say("model's end", rows, dtype)
    v = _run(p, s)
    _check_forward(s["x"], p["w1"], p["b1"], "gelu", None, v["h"], v["z"])
    _check_forward(v["h"], p["w2"], p["b2"], "none", s["x"], v["y"])
    _check_forward(v["y"], p["head"], None, "none", None, v["logits"])
    e = _check_logprobs(v["logits"], s["t"], 1.0, v["r"], 4)
    _check_logprob_gradient(v["logits"], s["t"], e, s["g"], s["w"], v["g2"])
    _check_distill(v["logits"], s["idx"], s["val"], 2.0, s["w"], v["loss"], v["g1"])
    assert not v["dl"][::6].any()
    _check_backward(v["dl"], v["y"], p["head"], None, "none", v["dy"], v["dhead"], None)
    _check_backward(v["dy"], v["h"], p["w2"], None, "none", v["dh"], v["dw2"], v["db2"])
    from cudeep_amd import ops
    dx, dw1, db1 = ops.linear16_backward(v["dh"], s["x"], p["w1"], v["z"], epilogue=_act_code("gelu"))
    _check_backward(v["dh"], s["x"], p["w1"], v["z"], "gelu", dx, dw1, db1)
    assert torch.equal(dx + v["dy"], v["dx"]) and torch.equal(dw1, v["dw1"]) and torch.equal(db1, v["db1"])
    assert not v["dx"][::6].any()


def test_a_step_in_a_graph():
    import torch
    p, s = _model("bf16"), _tokens(130, "bf16", 10)
    say("model's end in a graph")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _run(p, s)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = _run(p, s)
    for k in range(3):
        for name, value in _tokens(130, "bf16", 30 + 10 * k).items():
            s[name].copy_(value)
        want = _run(p, s)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name in want:
            if name == "r":
                assert all(torch.equal(a, b) for a, b in zip(held["r"], want["r"]))
            else:
                assert torch.equal(held[name], want[name]), name


def test_tokens_one_by_one():
    """A decoder's step: the log probabilities of one row are those of the batch, up to the order of the sums
    that different kernels take (each checked against 64 bits)."""
    from cudeep_amd import ops
    p, s = _model("bf16"), _tokens(9, "bf16", 10)
    for n in range(9):
        x, t = s["x"][n:n + 1], s["t"][n:n + 1].clamp_min(0)
        y = ops.linear16(ops.linear16(x, p["w1"], p["b1"], epilogue=_act_code("gelu")), p["w2"], p["b2"], residual=x)
        logits = ops.linear16(y, p["head"])
        _check_forward(y, p["head"], None, "none", None, logits)
        _check_logprobs(logits, t, 1.0, ops.token_logprobs(logits, t, entropy=True, top=4), 4)
