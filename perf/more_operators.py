"""The two ends of a model's last layers as cases that can be timed and compared: a Linear layer in
16 bits with bias, activation and residual in its epilogue, forward and backward, and what reads its
logits: the log probabilities of given tokens (with entropy and the likeliest alternatives, and their
gradient) and distillation from a teacher's top logits (loss and gradient).

A case is a dict of plain values; `prepare` makes its inputs, `run` is one pass: through
`cudeep_amd.ops` where `own` is set, else in elementary torch operations in 32 bits.  `exact` is the
same result in 64 bits.

Definitions.  Linear: z = x W^T + b, y = residual + act(z); its backward pass takes z as the forward
pass returned it, in x's type.  Rows of logits x with temperature T: l = log softmax(x / T) over the
vocabulary, the token's l_t (0 for a negative t), the entropy -sum p l, the k largest with the
lowest index first among equals.  Distillation: p = softmax(teacher / T) over a row's entries (those of
negative index do not count; without any the row's loss is 0), loss = sum p (log p - l_index), gradient
weight / T (softmax(x / T) - p at its indices).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
GELU_C, GELU_K = 0.7978845608, 0.044715


# ---- cases ---------------------------------------------------------------------------------

def linear(m, n, k, dtype, act="none", bias=True, residual=True, train=False, **more):
    return {"kind": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "act": act, "bias": bias,
            "residual": residual, "train": train, **more}


def logprob(rows, vocab, dtype, top=0, train=False, temperature=1.0, masked=False, **more):
    return {"kind": "logprob", "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
            "train": train, "temperature": temperature, "masked": masked, **more}


def distill(rows, vocab, dtype, count, temperature=1.0, grad=True, **more):
    return {"kind": "distill", "rows": rows, "vocab": vocab, "dtype": dtype, "count": count,
            "temperature": temperature, "grad": grad, **more}


def listed():
    return [
        # one token through a layer that adds to the residual stream: the weight's bytes and the call
        linear(1, 4096, 4096, "bf16", name="linear16_one_token"),
        # a handful of requests through a layer of odd sizes
        linear(37, 1000, 1200, "f16", act="gelu", name="linear16_ragged"),
        # a prompt of 4096 tokens through a layer with activation and residual
        linear(4096, 4096, 4096, "bf16", act="silu", name="linear16_4096"),
        # a training step of the benchmark's perceptron's first layer (784 -> 256)
        linear(8192, 256, 784, "f16", act="relu", residual=False, train=True, name="linear16_train_784"),
        # a training step of a layer on 8192 tokens: the largest
        linear(8192, 4096, 4096, "bf16", act="gelu", train=True, name="linear16_train_8192"),
        # one decoded token: its log probability and five alternatives
        logprob(1, 32000, "f32", top=5, masked=True, name="logprob_one_token"),
        # scoring a prompt of 2048 tokens over a large vocabulary, with alternatives
        logprob(2048, 131072, "bf16", top=8, temperature=0.7, name="logprob_prompt_2048"),
        # a policy's update on a ragged batch: log probabilities, entropies and their gradient
        logprob(1021, 50001, "f32", train=True, masked=True, name="logprob_train_ragged"),
        # the loss alone on a small batch, as an evaluation has it
        distill(16, 32000, "bf16", 16, grad=False, name="distill_eval_16"),
        # a distillation step on 4096 tokens: loss and gradient
        distill(4096, 65536, "bf16", 64, temperature=2.0, name="distill_train_4096"),
        # the same in single precision on a ragged batch
        distill(513, 50001, "f32", 20, name="distill_train_ragged"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm; two of four rounded to a multiple of 8 or 128,
    as layer sizes mostly are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice([1, 1, 8, 128])
    return max(lo, min(hi, (v + step // 2) // step * step))


def draw(rng):
    kind = rng.choice(["linear", "linear", "train", "logprob", "logprob_train", "distill"])
    if kind in ("linear", "train"):
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
        while m * n * k > 1 << 36:
            m = (m + 1) // 2
        return linear(m, n, k, rng.choice(["bf16", "f16"]), act=rng.choice(["none", "relu", "gelu", "silu"]),
                      bias=rng.random() < 0.7, residual=rng.random() < 0.6, train=kind == "train")
    rows, vocab = _log_int(rng, 1, 8192), _log_int(rng, 1000, 200000)
    while rows * vocab > 1 << 28:
        rows = (rows + 1) // 2
    dtype, temperature = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice([1.0, 1.0, 0.7, 2.0])
    if kind == "distill":
        return distill(rows, vocab, dtype, _log_int(rng, 1, 128), temperature=temperature,
                       grad=rng.random() < 0.75)
    return logprob(rows, vocab, dtype, top=0 if kind == "logprob_train" else rng.choice([0, 1, 5, 20]),
                   train=kind == "logprob_train", temperature=temperature, masked=rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def rnd(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=g) * scale

    dt, kind = DTYPES[case["dtype"]], case["kind"]
    s = {"case": dict(case)}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # activations with a few large channels; weights scaled by their fan-in
        s["x"] = (rnd(m, k) * rnd(1, k).mul(0.5).exp()).to(dt)
        s["w"] = rnd(n, k, scale=k ** -0.5).to(dt)
        s["b"] = rnd(n, scale=0.1).to(dt) if case["bias"] else None
        s["res"] = rnd(m, n).to(dt) if case["residual"] else None
        s["dy"] = rnd(m, n, scale=m ** -0.5).to(dt) if case["train"] else None
        return s
    rows, vocab = case["rows"], case["vocab"]
    # rows of their own sharpness, as a model's logits have them
    x = rnd(rows, vocab) * rnd(rows, 1).mul(0.3).exp().mul(2.0)
    usable = vocab
    if case.get("masked"):   # a vocabulary's unused end, and words that a grammar forbids
        usable = vocab - vocab // 16
        x[:, usable:] = -math.inf
        x[::3, 1:usable:2] = -math.inf
    s["x"] = x.to(dt)
    if kind == "logprob":
        t = torch.randint(0, (usable + 1) // 2, (rows,), device="cuda", generator=g) * 2
        t = t.clamp_max(usable - 1) // 2 * 2
        if rows > 8:   # the padding of a ragged batch
            t[::8] = -100
        s["t"] = t
        if case["train"]:
            s["g"], s["gh"] = rnd(rows), rnd(rows, scale=0.01)
        return s
    k = case["count"]
    # what a teacher of similar logits thinks likely, its entries in no order, some rows' lists shorter
    v = (rnd(rows, k) * 2.0 + 4.0).to(dt)
    i = torch.randint(0, vocab, (rows, k), device="cuda", generator=g)
    short = torch.randint(0, k + 1, (rows, 1), device="cuda", generator=g)
    cut = (torch.arange(rows, device="cuda") % 4 == 1)[:, None] & (torch.arange(k, device="cuda") >= short)
    s["i"], s["v"] = torch.where(cut, torch.full_like(i, -1), i), v
    s["wt"] = torch.rand(rows, device="cuda", generator=g) / rows if case["grad"] else None
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _run_own(s):
    from cudeep_amd import ops
    from cudeep_amd import _lib as L
    acts = {"none": L.EPI_NONE, "relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU}
    c = s["case"]
    if c["kind"] == "linear":
        act = acts[c["act"]]
        if not c["train"]:
            return ops.linear16(s["x"], s["w"], s["b"], epilogue=act, residual=s["res"])
        y, z = ops.linear16(s["x"], s["w"], s["b"], epilogue=act, residual=s["res"], keep=True)
        dx, dw, db = ops.linear16_backward(s["dy"], s["x"], s["w"], z, epilogue=act, bias=c["bias"])
        return (y, z, dx, dw, db) if c["bias"] else (y, z, dx, dw)
    temperature = c["temperature"]
    if c["kind"] == "logprob":
        r = ops.token_logprobs(s["x"], s["t"], temperature=temperature, entropy=True, top=c["top"])
        if c["train"]:
            dx = ops.token_logprobs_backward(s["g"], s["x"], s["t"], r.stats, entropy=r.entropy,
                                             grad_entropy=s["gh"], temperature=temperature)
            return r.logprob, r.entropy, dx
        if c["top"]:
            return r.logprob, r.entropy, r.top_logprob, r.top_index
        return r.logprob, r.entropy
    return ops.distill_loss(s["x"], s["i"], s["v"], temperature=temperature, weight=s["wt"])


def _act(v, act):
    if act == "relu":
        return v.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(GELU_C * (v + GELU_K * v * v * v)))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        t = torch.tanh(GELU_C * (z + GELU_K * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_C * (1.0 + 3.0 * GELU_K * z * z)
    if act == "silu":
        p = 1.0 / (1.0 + torch.exp(-z))
        return p * (1.0 + z * (1.0 - p))
    return torch.ones_like(z)


def _plain_linear(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, c["act"])
    if s["res"] is not None:
        y = y + s["res"].float()
    if not c["train"]:
        return y.to(dt)
    z = z.to(dt)   # an output, and what the backward pass takes
    dz = s["dy"].float() * _act_grad(z.float(), c["act"])
    out = y.to(dt), z, (dz @ w).to(dt), (dz.t() @ x).to(dt)
    return (*out, dz.sum(0).to(dt)) if c["bias"] else out


def _order_keys(x):
    """An int64 for each value of a float32 matrix that orders a row by value, then lowest index."""
    u = (x + 0.0).view(torch.int32)
    u = u ^ ((u >> 31) & 0x7FFFFFFF)
    return (u.long() << 32) + (0x7FFFFFFF - torch.arange(x.shape[1], device=x.device))


def _log_softmax(x, temperature):
    """(log softmax(x / T), softmax(x / T)) of rows with at least one finite value."""
    d = (x - x.amax(-1, keepdim=True)) / temperature
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    return d - torch.log(total), e / total


def _times(p, l):
    """p l where p is not 0."""
    return torch.where(p > 0, p * l, torch.zeros_like(p))


def _plain_logprob(s):
    c, t = s["case"], s["t"]
    x = s["x"].float()
    l, p = _log_softmax(x, c["temperature"])
    there = t >= 0
    at = t.clamp_min(0)[:, None]
    lp = torch.where(there, l.gather(1, at)[:, 0], torch.zeros_like(l[:, 0]))
    h = -_times(p, l).sum(-1)
    if c["train"]:
        g = torch.where(there, s["g"], torch.zeros_like(lp))[:, None]
        dx = -p * g
        dx = dx.scatter_add(1, at, g)
        dx = dx - s["gh"][:, None] * _times(p, l + h[:, None])
        return lp, h, (dx / c["temperature"]).to(s["x"].dtype)
    if not c["top"]:
        return lp, h
    index = 0x7FFFFFFF - (torch.topk(_order_keys(x), c["top"], dim=1).values & 0xFFFFFFFF)
    return lp, h, l.gather(1, index), index


def _plain_distill(s):
    c, i = s["case"], s["i"]
    x, there, at = s["x"].float(), i >= 0, i.clamp_min(0)
    l, q = _log_softmax(x, c["temperature"])
    v = torch.where(there, s["v"].float() / c["temperature"], torch.full_like(i, -math.inf, dtype=torch.float32))
    top = v.amax(-1, keepdim=True)
    e = torch.where(there, torch.exp(v - torch.where(top > -math.inf, top, torch.zeros_like(top))), torch.zeros_like(v))
    total = e.sum(-1, keepdim=True)
    some = total > 0
    p = torch.where(some, e / total, torch.zeros_like(e))
    logp = torch.where(there & some, v - top - torch.log(total), torch.zeros_like(v))
    loss = (p * (logp - l.gather(1, at))).sum(-1)
    if s["wt"] is None:
        return loss
    f = (s["wt"][:, None] / c["temperature"]) * some
    return loss, (f * q).scatter_add(1, at, -f * p).to(s["x"].dtype)


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    return _plain_linear(s) if kind == "linear" else _plain_logprob(s) if kind == "logprob" else _plain_distill(s)


# ---- work and the result in 64 bits --------------------------------------------------------------

def work(case):
    e = BYTES[case["dtype"]]
    if case["kind"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        b = n if case["bias"] else 0
        values = m * k + n * k + b + m * n * (2 if case["residual"] else 1)
        if case["train"]:   # dy and z, and the gradients
            values += 2 * m * n + m * k + n * k + b
        return {"bytes": values * e, "flops": (6 if case["train"] else 2) * m * n * k}
    x = case["rows"] * case["vocab"]
    if case["kind"] == "logprob":
        out = case["rows"] * (8 + 8 + 12 * case["top"])
        if case["train"]:
            return {"bytes": 2 * x * e + out + 8 * case["rows"], "flops": 14 * x}
        return {"bytes": x * e + out, "flops": 6 * x}
    lists = case["rows"] * case["count"] * (8 + e)
    if case["grad"]:
        return {"bytes": 2 * x * e + lists + 8 * case["rows"], "flops": 8 * x}
    return {"bytes": x * e + lists + 4 * case["rows"], "flops": 4 * x}


def _exact_linear(s):
    case = s["case"]
    x, w = s["x"].double(), s["w"].double()
    z = torch.addmm(s["b"].double(), x, w.t()) if case["bias"] else x @ w.t()
    zk = z.to(DTYPES[case["dtype"]]).double()   # what the backward pass is given
    up = 2.0 * GELU_C * (z + GELU_K * z ** 3)
    if case["act"] == "gelu":   # 0.5 (1 + tanh u) = 1 / (1 + exp(-2u))
        y = z * torch.sigmoid(up)
        p = torch.sigmoid(2.0 * GELU_C * (zk + GELU_K * zk ** 3))
        slope = p + 2.0 * zk * p * (1.0 - p) * GELU_C * (1.0 + 3.0 * GELU_K * zk ** 2)
    elif case["act"] == "silu":
        y = z * torch.sigmoid(z)
        p = torch.sigmoid(zk)
        slope = p + zk * p * (1.0 - p)
    elif case["act"] == "relu":
        y, slope = torch.where(z > 0, z, 0.0), torch.where(zk > 0, 1.0, 0.0).double()
    else:
        y, slope = z, torch.ones_like(z)
    if case["residual"]:
        y = s["res"].double() + y
    if not case["train"]:
        return y
    dz = s["dy"].double() * slope
    out = y, z, dz @ w, dz.t().contiguous() @ x
    return (*out, dz.sum(0)) if case["bias"] else out


def _exact_logprob(s):
    case = s["case"]
    u = s["x"].double() / case["temperature"]
    there = s["t"] >= 0
    at = s["t"].clamp_min(0)[:, None]
    norm = torch.logsumexp(u, -1, keepdim=True)
    lp = torch.where(there, (u.gather(1, at) - norm)[:, 0], 0.0)
    p = torch.exp(u - norm)
    mean = torch.where(p > 0, p * u, 0.0).sum(-1, keepdim=True)   # the mean of u: H = norm - mean
    h = (norm - mean)[:, 0]
    if case["train"]:
        g = torch.where(there, s["g"].double(), 0.0)[:, None]
        # d l_t / du = 1 at t - p, dH / du = p (mean - u)
        dx = torch.where(p > 0, s["gh"].double()[:, None] * p * (mean - u), 0.0) - g * p
        return lp, h, dx.scatter_add_(1, at, g) / case["temperature"]
    if not case["top"]:
        return lp, h
    return lp, h, torch.topk(u, case["top"], dim=1).values - norm, None


def _exact_distill(s):
    case = s["case"]
    u = s["x"].double() / case["temperature"]
    there, at = s["i"] >= 0, s["i"].clamp_min(0)
    norm = torch.logsumexp(u, -1, keepdim=True)
    v = torch.where(there, s["v"].double() / case["temperature"], -math.inf)
    some = there.any(-1, keepdim=True)
    p = torch.where(some, torch.nn.functional.pad(v, (0, 1), value=-1e300).softmax(-1)[:, :-1], 0.0)
    cross = (p * (norm - u.gather(1, at))).sum(-1)
    loss = torch.special.xlogy(p, p).sum(-1) + cross
    if not case["grad"]:
        return loss
    f = s["wt"].double()[:, None] * some / case["temperature"]
    return loss, torch.exp(u - norm).mul_(f).scatter_add_(1, at, -f * p)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    return _exact_linear(s) if kind == "linear" else _exact_logprob(s) if kind == "logprob" else _exact_distill(s)
