"""The operators that stand around a Linear layer in training and serving, as cases that can be
timed and compared: layer norm with its backward pass, products of 8-bit floating-point operands
with a scale for each block of 128, and activations kept in 8 bits for the backward pass.

A case is a dict of plain values; `prepare` makes its inputs (and the quantised weight or the
checkpoint that a program would hold), `run` is one pass: through `cudeep_amd.ops` where `own` is
set, else in elementary torch operations in 32 bits.  `exact` is the same result in 64 bits.

The 8-bit format: e4m3 values (largest 448) and, for each 128 columns of a row (activations) or each
128 x 128 tile (weights), a scale 2^e with the least e in [-117, 120] for which the block's largest
magnitude is at most 448 * 2^e (1 for a block of zeros).
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 128
GELU_C, GELU_K = 0.7978845608, 0.044715


# ---- cases ---------------------------------------------------------------------------------

def norm(rows, dim, dtype, train, affine=True, **more):
    return {"kind": "norm", "rows": rows, "dim": dim, "dtype": dtype, "train": train,
            "affine": affine, **more}


def linear(m, n, k, dtype, scales="e8m0", bias=True, act="none", **more):
    return {"kind": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "scales": scales,
            "bias": bias, "act": act, **more}


def product(m, n, k, dtype, scales="e8m0", **more):
    return {"kind": "product", "m": m, "n": n, "k": k, "dtype": dtype, "scales": scales, **more}


def store(rows, cols, dtype, **more):
    return {"kind": "store", "rows": rows, "cols": cols, "dtype": dtype, **more}


def gelu(rows, cols, dtype, **more):
    return {"kind": "gelu", "rows": rows, "cols": cols, "dtype": dtype, **more}


def wgrad(m, n, k, dtype, bias=True, **more):
    return {"kind": "wgrad", "m": m, "n": n, "k": k, "dtype": dtype, "bias": bias, **more}


def listed():
    return [
        # one token of a served model: launch and latency count
        norm(1, 4096, "bf16", False, name="norm_one_token"),
        # a training step's norm on 8192 tokens: forward, gradients of input, weight and bias
        norm(8192, 4096, "bf16", True, name="norm_train_8192"),
        # the same in single precision on a ragged last batch, a width that fills no whole wave
        norm(4099, 1000, "f32", True, name="norm_train_ragged"),
        # one token through a layer whose weight is held in 8 bits: the weight's bytes are the floor
        linear(1, 4096, 4096, "bf16", name="linear8_one_token"),
        # a handful of requests through a layer of odd sizes, weight scales as published weights have them
        linear(37, 1000, 1200, "f16", scales="f32", act="gelu", name="linear8_ragged"),
        # a layer on 4096 tokens of a batch or prompt, activations quantised on the way in
        linear(4096, 4096, 4096, "bf16", act="gelu", name="linear8_4096"),
        # a long prompt, operands already in 8 bits: the largest product
        product(8192, 8192, 4096, "bf16", scales="f32", name="product8_8192"),
        # activations stored in 8 bits and restored for a recomputation
        store(8192, 4096, "bf16", name="store8_8192"),
        # the activation between two layers, its input kept in 8 bits, and its backward pass
        gelu(8192, 4096, "bf16", name="gelu8_8192"),
        # the weight gradient of the benchmark's perceptron (784 -> 256) from an 8-bit input
        wgrad(8192, 256, 784, "f32", name="wgrad8_perceptron"),
        # the weight gradient of a layer on 8192 tokens
        wgrad(8192, 4096, 4096, "bf16", bias=False, name="wgrad8_8192"),
        # a small ragged layer on a few rows
        wgrad(64, 250, 333, "f32", name="wgrad8_small"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread evenly over the logarithm; two of four rounded to a multiple of 8 or 128,
    as layer sizes mostly are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice([1, 1, 8, 128])
    return max(lo, min(hi, (v + step // 2) // step * step))


def draw(rng):
    kind = rng.choice(["norm", "norm", "linear", "linear", "product", "store", "gelu", "wgrad", "wgrad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "norm":
        rows, dim = _log_int(rng, 1, 32768), _log_int(rng, 16, 16384)
        while rows * dim > 1 << 25:
            rows = (rows + 1) // 2
        return norm(rows, dim, dtype, rng.random() < 0.6, affine=rng.random() < 0.8)
    if kind in ("linear", "product"):
        m, n, k = _log_int(rng, 1, 8192), _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
        while m * n * k > 1 << 37:
            m = (m + 1) // 2
        scales = rng.choice(["e8m0", "f32"])
        if kind == "product":
            return product(m, n, k, dtype, scales=scales)
        return linear(m, n, k, dtype, scales=scales, bias=rng.random() < 0.7,
                      act=rng.choice(["none", "relu", "gelu", "silu"]))
    if kind in ("store", "gelu"):
        rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 16, 16384)
        while rows * cols > 1 << 25:
            rows = (rows + 1) // 2
        return (store if kind == "store" else gelu)(rows, cols, dtype)
    m, n, k = _log_int(rng, 1, 16384), _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
    while m * n * k > 1 << 36:
        m = (m + 1) // 2
    return wgrad(m, n, k, dtype, bias=rng.random() < 0.7)


# ---- the 8-bit format in elementary operations ------------------------------------------------

def _pow2(e):
    """2^e in float32 from an int32 tensor of exponents (-126 .. 127)."""
    return ((e + 127) << 23).view(torch.float32)


def _blocks(x):
    """[rows, cols] -> [rows, blocks, 128], padded with zeros."""
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, -cols % BLOCK)).view(rows, -1, BLOCK)


def _exponents(amax):
    """The scale's exponent of blocks with these largest magnitudes: 448 = 0.875 * 2^9."""
    frac, e = torch.frexp(amax)
    e = torch.where(frac <= 0.875, e - 9, e - 8).clamp(-117, 120).to(torch.int32)
    return torch.where(amax > 0, e, torch.zeros_like(e))


def _quantize_rows(x):
    """(e4m3 values, exponents [rows, blocks]) with a scale for each 128 columns of a row."""
    b = _blocks(x.float())
    mag = b.abs()
    e = _exponents(torch.where(mag < math.inf, mag, torch.zeros_like(mag)).amax(-1))
    q = (b * _pow2(-e).unsqueeze(-1)).view(x.shape[0], -1)[:, : x.shape[1]]
    q = torch.where(q.abs() < math.inf, q, torch.full_like(q, math.nan))
    return q.to(torch.float8_e4m3fn), e


def _quantize_tiles(w):
    """(e4m3 values, exponents [row tiles, blocks]) with a scale for each 128 x 128 tile."""
    rows, cols = w.shape
    p = torch.nn.functional.pad(w.float(), (0, -cols % BLOCK, 0, -rows % BLOCK))
    t = p.view(p.shape[0] // BLOCK, BLOCK, p.shape[1] // BLOCK, BLOCK)
    e = _exponents(t.abs().amax((1, 3)))
    q = (t * _pow2(-e)[:, None, :, None]).view(p.shape)[:rows, :cols]
    return q.contiguous().to(torch.float8_e4m3fn), e


def _scale(e, kind):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu) if kind == "e8m0" else _pow2(e)


def _scale_values(s):
    """A scale tensor as float32."""
    if s.dtype == torch.float32:
        return s
    return _pow2(s.view(torch.uint8).to(torch.int32) - 127)


def _restore(q, s):
    """The float32 values of 8-bit values with the scale of each 128 columns of a row."""
    rows, cols = q.shape
    return (_blocks(q.float()) * _scale_values(s).unsqueeze(-1)).view(rows, -1)[:, :cols]


def _restore_tiles(q, s):
    """The same with the scale of each 128 x 128 tile."""
    rows, cols = q.shape
    full = _scale_values(s).repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return q.float() * full


# ---- inputs ----------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def rnd(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=g) * scale

    dt, kind = DTYPES[case["dtype"]], case["kind"]
    s = {"case": dict(case)}
    if kind == "norm":
        rows, dim = case["rows"], case["dim"]
        # rows of their own mean and spread, as a residual stream has them
        x = rnd(rows, dim) * rnd(rows, 1).mul(0.5).exp() + rnd(rows, 1)
        s["x"] = x.to(dt)
        s["w"] = (1.0 + rnd(dim, scale=0.2)).to(dt) if case["affine"] else None
        s["b"] = rnd(dim, scale=0.2).to(dt) if case["affine"] else None
        s["dy"] = rnd(rows, dim).to(dt) if case["train"] else None
    elif kind in ("linear", "product"):
        m, n, k = case["m"], case["n"], case["k"]
        # activations with a few large channels; weights scaled by their fan-in
        x = (rnd(m, k) * rnd(1, k).mul(0.5).exp()).to(dt)
        q, e = _quantize_tiles(rnd(n, k, scale=k ** -0.5))
        s["wq"], s["ws"] = q, _scale(e, case["scales"])
        if case["scales"] == "f32":   # scales that are no powers of two
            s["ws"] = s["ws"] * (1.0 + torch.rand(e.shape, device="cuda", generator=g))
        if kind == "linear":
            s["x"] = x
            s["bias"] = rnd(n, scale=0.1) if case["bias"] else None
        else:
            s["xq"], e = _quantize_rows(x)
            s["xs"] = _scale(e, case["scales"])
            if case["scales"] == "f32":
                s["xs"] = s["xs"] * (1.0 + torch.rand(e.shape, device="cuda", generator=g))
    elif kind == "store":
        s["x"] = (rnd(case["rows"], case["cols"]) * rnd(1, case["cols"]).mul(0.5).exp()).to(dt)
    elif kind == "gelu":
        s["z"] = rnd(case["rows"], case["cols"], scale=1.5).to(dt)
        s["dy"] = rnd(case["rows"], case["cols"]).to(dt)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["dz"] = (rnd(m, n) * m ** -0.5).to(dt)
        s["xq"], e = _quantize_rows(rnd(m, k) * rnd(1, k).mul(0.5).exp())
        s["xs"] = _scale(e, "e8m0")
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _run_own(s):
    from cudeep_amd import ops
    from cudeep_amd import _lib as L
    acts = {"none": L.EPI_NONE, "relu": L.EPI_RELU, "gelu": L.EPI_GELU, "silu": L.EPI_SILU}
    c = s["case"]
    kind, dt = c["kind"], DTYPES[c["dtype"]]
    if kind == "norm":
        if not c["train"]:
            return ops.layer_norm(s["x"], s["w"], s["b"])
        y, mean, rstd = ops.layer_norm(s["x"], s["w"], s["b"], stats=True)
        dx, dw, db = ops.layer_norm_backward(s["dy"], s["x"], mean, rstd, s["w"],
                                             params=c["affine"])
        return (y, dx, dw, db) if c["affine"] else (y, dx)
    if kind == "linear":
        w = ops.Block8(s["wq"], s["ws"], 128)
        return ops.linear8(s["x"], w, s["bias"], epilogue=acts[c["act"]])
    if kind == "product":
        return ops.gemm8(ops.Block8(s["xq"], s["xs"], 1), ops.Block8(s["wq"], s["ws"], 128), dtype=dt)
    if kind == "store":
        return ops.dequantize8(ops.quantize8(s["x"]), dtype=dt)
    if kind == "gelu":
        y, kept = ops.activation8(s["z"], L.EPI_GELU)
        return y, ops.activation_backward8(s["dy"], kept, L.EPI_GELU)
    dw, db = ops.linear_weight_grad8(s["dz"], ops.Block8(s["xq"], s["xs"], 1), bias=c["bias"])
    return (dw, db) if c["bias"] else dw


def _act(v, act):
    if act == "relu":
        return v.clamp_min(0.0)
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.tanh(GELU_C * (v + GELU_K * v * v * v)))
    if act == "silu":
        return v * torch.sigmoid(v)
    return v


def _gelu_grad(z):
    t = torch.tanh(GELU_C * (z + GELU_K * z * z * z))
    return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * GELU_C * (1.0 + 3.0 * GELU_K * z * z)


def _run_plain(s):
    c = s["case"]
    kind, dt = c["kind"], DTYPES[c["dtype"]]
    if kind == "norm":
        x = s["x"].float()
        mean = x.mean(-1, keepdim=True)
        d = x - mean
        rstd = torch.rsqrt((d * d).mean(-1, keepdim=True) + 1e-5)
        xh = d * rstd
        w = s["w"].float() if c["affine"] else None
        y = (xh * w + s["b"].float() if c["affine"] else xh).to(dt)
        if not c["train"]:
            return y
        dy = s["dy"].float()
        g = dy * w if c["affine"] else dy
        dx = (rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))).to(dt)
        if not c["affine"]:
            return y, dx
        return y, dx, (dy * xh).sum(0).to(dt), dy.sum(0).to(dt)
    if kind == "linear":
        q, e = _quantize_rows(s["x"])
        y = _restore(q, _pow2(e)) @ _restore_tiles(s["wq"], s["ws"]).t()
        if s["bias"] is not None:
            y = y + s["bias"]
        return _act(y, c["act"]).to(dt)
    if kind == "product":
        return (_restore(s["xq"], s["xs"]) @ _restore_tiles(s["wq"], s["ws"]).t()).to(dt)
    if kind == "store":
        q, e = _quantize_rows(s["x"])
        return _restore(q, _pow2(e)).to(dt)
    if kind == "gelu":
        z = s["z"].float()
        q, e = _quantize_rows(z)
        return _act(z, "gelu").to(dt), (s["dy"].float() * _gelu_grad(_restore(q, _pow2(e)))).to(dt)
    dz = s["dz"].float()
    dw = dz.t() @ _restore(s["xq"], s["xs"])
    return (dw, dz.sum(0)) if c["bias"] else dw


def run(s):
    return _run_own(s) if own else _run_plain(s)


# ---- work and the result in 64 bits --------------------------------------------------------------

def work(case):
    e, kind = BYTES[case["dtype"]], case["kind"]
    if kind == "norm":
        x = case["rows"] * case["dim"]
        p = 2 * case["dim"] * e if case["affine"] else 0
        if not case["train"]:
            return {"bytes": 2 * x * e + p, "flops": 8 * x}
        return {"bytes": 4 * x * e + 2 * p, "flops": 22 * x}
    if kind in ("linear", "product"):
        m, n, k = case["m"], case["n"], case["k"]
        es = 1 if case["scales"] == "e8m0" else 4
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        a = m * k * e if kind == "linear" else m * k + m * kb * es
        bias = 4 * n if case.get("bias") else 0
        return {"bytes": a + n * k + nb * kb * es + bias + m * n * e, "flops": 2 * m * n * k}
    if kind == "store":
        x = case["rows"] * case["cols"]
        return {"bytes": 2 * x * e, "flops": 4 * x}
    if kind == "gelu":
        x = case["rows"] * case["cols"]
        return {"bytes": 4 * x * e, "flops": 40 * x}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": m * n * e + m * k + m * -(-k // BLOCK) + 4 * n * k + (4 * n if case["bias"] else 0),
            "flops": 2 * m * n * k}


def _exact_rows(x):
    """Values of x (float64) after the 8-bit rounding, from the definition of the format: each
    value is rounded to a multiple of 2^(its exponent - 3), no finer than 2^-9, of its block's
    scale, ties to even."""
    rows, cols = x.shape
    out = torch.zeros((rows, -(-cols // BLOCK) * BLOCK), dtype=torch.float64, device=x.device)
    out[:, :cols] = x
    out = out.view(rows, -1, BLOCK)
    top = out.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -200) / 448.0))
    # the logarithm may be off by its own rounding where top is at a power of two times 448
    e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e).clamp(-117, 120)
    s = torch.where(top > 0, torch.exp2(e), torch.ones_like(e))
    v = out / s
    _, ve = torch.frexp(v)
    step = torch.exp2((ve.to(torch.float64) - 1).clamp_min(-6.0) - 3)
    return (torch.round(v / step) * step * s).view(rows, -1)[:, :cols]


def _exact_scale(s):
    return s.double() if s.dtype == torch.float32 else torch.exp2(s.view(torch.uint8).double() - 127.0)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, -1, keepdim=True, correction=0)
        xh = (x - mean) / torch.sqrt(var + 1e-5)
        w = s["w"].double() if case["affine"] else torch.ones((), device="cuda", dtype=torch.float64)
        b = s["b"].double() if case["affine"] else torch.zeros((), device="cuda", dtype=torch.float64)
        y = xh * w + b
        if not case["train"]:
            return y
        dy, dim = s["dy"].double(), case["dim"]
        g = dy * w
        dx = (dim * g - g.sum(-1, keepdim=True) - xh * (g * xh).sum(-1, keepdim=True)) \
            / (dim * torch.sqrt(var + 1e-5))
        if not case["affine"]:
            return y, dx
        return y, dx, torch.einsum("rd,rd->d", dy, xh), dy.sum(0)
    if kind in ("linear", "product"):
        n, k = case["n"], case["k"]
        rows = torch.arange(n, device="cuda") // BLOCK
        cols = torch.arange(k, device="cuda") // BLOCK
        w = s["wq"].double() * _exact_scale(s["ws"])[rows][:, cols]
        if kind == "product":
            return (s["xq"].double() * _exact_scale(s["xs"])[:, cols]) @ w.t()
        y = _exact_rows(s["x"].double()) @ w.t()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        if case["act"] == "relu":
            return torch.where(y > 0, y, torch.zeros_like(y))
        if case["act"] == "gelu":   # 0.5 (1 + tanh u) = 1 / (1 + exp(-2u))
            return y / (1.0 + torch.exp(-2.0 * GELU_C * (y + GELU_K * y ** 3)))
        return y / (1.0 + torch.exp(-y)) if case["act"] == "silu" else y
    if kind == "store":
        return _exact_rows(s["x"].double())
    if kind == "gelu":
        z, zh = s["z"].double(), _exact_rows(s["z"].double())
        p = 1.0 / (1.0 + torch.exp(-2.0 * GELU_C * (zh + GELU_K * zh ** 3)))
        slope = p + 2.0 * zh * p * (1.0 - p) * GELU_C * (1.0 + 3.0 * GELU_K * zh ** 2)
        return z / (1.0 + torch.exp(-2.0 * GELU_C * (z + GELU_K * z ** 3))), s["dy"].double() * slope
    dz = s["dz"].double()
    cols = torch.arange(case["k"], device="cuda") // BLOCK
    dw = dz.t().contiguous() @ (s["xq"].double() * _exact_scale(s["xs"])[:, cols])
    return (dw, dz.sum(0)) if case["bias"] else dw
